"""Paged attention through qmr_encode_static: the ranges that it leaves in the
scratch, plans cut to the scratch, and launches after it that need zeros there."""
from __future__ import annotations

import numpy as np
import pytest

import qmr
from attention_cases import Batch, attend, attend64, check_attend, from_half, make_pool
from helpers import assert_gate
from test_zz_no_alloc import _case, _launch

pytestmark = pytest.mark.gpu


def inputs(kind, batch, heads, kv_heads, dim, seed):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((batch.tokens, heads, dim)).astype(np.float32)
    return q, *make_pool(batch, kv_heads, dim, kind, rng)


@pytest.fixture()
def fresh():
    g = qmr.Gpu("aligned")
    yield g
    assert g.workspace_bytes() == 0, "the static entry allocated"
    g.close()


# Launches that add into slots or count arrivals, which have to be zero.
AFTER = [("plain", (0, 0), (5120, 17408, 3)), ("plain", (-2, 0), (17408, 5120, 2)), ("dense", (-5, 408), (17408, 5120, 4)),
         ("mlp", (0, 0), (4096, 2048, 3))]


@pytest.mark.parametrize("form,plan,shape", AFTER)
def test_ranges_in_the_scratch_and_a_launch_that_needs_zeros(gpu, fresh, form, plan, shape):
    batch = Batch([1, 1], [3000, 900], 64)
    q, k, v = inputs("f16", batch, 12, 2, 128, 1)
    want, bound = attend64(q, from_half(k, "f16"), from_half(v, "f16"), batch, 0.125)
    name, arrays, params, product = _case(np.random.default_rng(3), form, *shape)
    for turn in range(2):
        got = attend(fresh, "f16", q, k, v, batch, 0.125, static=True)
        assert np.array_equal(got, attend(gpu, "f16", q, k, v, batch, 0.125)), turn
        check_attend(got, want, bound, f"turn {turn}")
        y, kernel = _launch(fresh, name, arrays, params, shape[0], shape[2], True, plan)
        ref, ref_kernel = _launch(gpu, name, arrays, params, shape[0], shape[2], False, plan)
        assert kernel == ref_kernel and np.array_equal(y.view(np.uint32), ref.view(np.uint32)), (turn, kernel)
        assert_gate(y, product, f"{name} after attention, turn {turn}")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_a_plan_is_cut_to_the_scratch(gpu, fresh, kind):
    # 512 tokens of 24/4 heads of 256 over 16513 keys: qmr_encode's ranges take more
    # than the scratch.
    new, length = 512, 16513
    batch = Batch([new], [length], 64)
    q, k, v = inputs(kind, batch, 24, 4, 256, 2)
    other = qmr.Gpu("aligned")
    try:
        attend(other, kind, q, k, v, batch, 0.0625)
        assert other.workspace_bytes() > qmr.STATIC_SCRATCH_BYTES
    finally:
        other.close()
    last = Batch([3], [length], 64)
    assert np.array_equal(last.table, batch.table)
    want, bound = attend64(q[-3:], from_half(k, kind), from_half(v, kind), last, 0.0625)
    # The planner's choice, and more ranges than fit.
    for plan in ((0, 0), (-7, 16040), (-7, 128040)):
        fresh.set_gemv_plan(*plan)
        got = attend(fresh, kind, q, k, v, batch, 0.0625, static=True)
        check_attend(got[-3:], want, bound, f"plan {plan}")
        assert np.isfinite(got).all()
