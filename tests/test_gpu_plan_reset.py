"""A plan that a test forces on the shared device handle ends with the test."""
import numpy as np
import pytest

from qmr import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("leaves", [True, False])
def test_a_forced_plan_does_not_reach_the_next_test(gpu, leaves):
    # Of a product of eight columns, which takes the wide kernel unless a plan
    # for another kernel is in force.
    m = synth.q4_bf16_matrix(512, 512, synth.DEFAULT_SEED, "reset")
    bufs = [*(gpu.upload_bytes(a) for a in (m.w, m.s, m.b)), gpu.upload_f32(np.ones(8 * 512, np.float32)),
            gpu.alloc_f32(8 * 512)]
    gpu.dispatch("matmul_affine_wide_bf16", bufs, [512, 512, 4, 64, 8])
    assert gpu.last_hip_kernel().startswith("wide_mfma_kernel")
    if leaves:
        gpu.set_gemv_plan(-7, 0)
