"""attn_linear and sample_logits through the static scratch: what does not fit it,
and launches behind them that need zeros there."""
import numpy as np
import pytest

import qmr
from helpers import assert_gate
from linear_cases import Linear
from sample_cases import Sample
from test_gpu_linear import CHUNKS, TOKENS
from test_zz_no_alloc import _case, _launch
from test_zz_no_alloc_attention import AFTER

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts, chunks", [([33], True), ([223], True), ([224], False), ([200, 1, 130], False)])
def test_64_heads_of_128(gpu, counts, chunks):
    """Two states that passes would hand on are 8.06 MB. Seven chunks, of 1.1 MB each,
    fit the 8 MB of the scratch in one pass, with qmr_encode's bits (a launch counts
    tokens / 32 and one more for every sequence); more tokens go one after the
    other, and are right as well."""
    case = Linear(counts, 16, 64, 128, 128)
    out, after = case.check(gpu, CHUNKS)
    got, state = case.check(gpu, CHUNKS if chunks else TOKENS, static=True)
    assert gpu.last_hip_kernel() == ("linear_scan_kernel" if chunks else "attn_linear_tokens_kernel")
    if chunks:
        assert np.array_equal(got, out) and np.array_equal(state, after)


@pytest.fixture()
def fresh():
    g = qmr.Gpu("aligned")
    yield g
    assert g.workspace_bytes() == 0, "the static entry allocated"
    g.close()


@pytest.mark.parametrize("form,plan,shape", AFTER)
@pytest.mark.parametrize("which", ["attention", "draw"])
def test_launches_that_need_zeros_behind_them(gpu, fresh, which, form, plan, shape):
    if which == "attention":
        case = Linear([700, 40], 8, 16, 128, 128)
    else:
        case = Sample(np.random.default_rng(5).standard_normal((60, 30000)), 1.0, 300, 0.9)
    want = case.run(gpu)
    name, arrays, params, product = _case(np.random.default_rng(3), form, *shape)
    for turn in range(2):
        for got, expected in zip(case.run(fresh, static=True), want):
            assert np.array_equal(got, expected), turn
        y, kernel = _launch(fresh, name, arrays, params, shape[0], shape[2], True, plan)
        ref, ref_kernel = _launch(gpu, name, arrays, params, shape[0], shape[2], False, plan)
        assert kernel == ref_kernel and np.array_equal(y.view(np.uint32), ref.view(np.uint32)), (turn, kernel)
        assert_gate(y, product, f"{name} after {which}, turn {turn}")
