"""attn_paged where a mask, a missing page or a number that is not finite decides
what a row is."""
import numpy as np
import pytest

from attention_cases import Batch, attend, attend64, check_attend, from_half, make_pool, to_half

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]
# The planner's choice, and each kernel with and without key ranges.
PLANS = [0, 16001, 16003, 128001, 128002]


def under_plans(gpu, call):
    """(plan, call()) under each plan."""
    out = []
    try:
        for plan in PLANS:
            gpu.set_gemv_plan(-7, plan)
            out.append((plan, call()))
    finally:
        gpu.set_gemv_plan(0, 0)
    return out


def inputs(kind, batch, heads, kv_heads, dim, seed):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((batch.tokens, heads, dim)).astype(np.float32)
    return q, *make_pool(batch, kv_heads, dim, kind, rng)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30])
def test_windows_longer_than_every_position(gpu, kind, window):
    # With more new tokens than positions, whose first ones are negative.
    batch = Batch([5, 3, 40, 1], [2, 0, 30, 70], 32)
    q, k, v = inputs(kind, batch, 6, 2, 64, 1)
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, 0.125, window=window)
    assert np.abs(want[3:5]).max() > 0.1 and (want[:3] == 0).all()
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.125, window=window)):
        check_attend(got, want, bound, f"plan {plan}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [2e-40, 1e-41, 1e-44])
def test_queries_near_zero(gpu, kind, size):
    # Scores that vanish, beside keys that a row does not see: plain means.
    batch = Batch([1, 3, 40], [20, 37, 200], 32)
    q, k, v = inputs(kind, batch, 4, 2, 64, 3)
    q = (q * size).astype(np.float32)
    assert (np.abs(q).reshape(batch.tokens, -1).max(axis=1) > 0).all()
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, 0.5)
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.5)):
        check_attend(got, want, bound, f"plan {plan}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [3, 140])
def test_queries_that_see_nothing_are_zero_whatever_they_hold(gpu, kind, new):
    # All pages of the first sequence are past the pool; the second has no cache.
    batch = Batch([new, 2, 1], [300, 0, 40], 32, dropped=tuple((0, c) for c in range(10)))
    q, k, v = inputs(kind, batch, 4, 2, 64, 2)
    clean = q.copy()
    q[:new:2, :, 5], q[1:new:2, :, 6] = np.nan, np.inf
    q[new:new + 2, 1, 0] = np.nan
    want, bound = attend64(clean, from_half(k, kind), from_half(v, kind), batch, 0.125)
    assert (want[:new + 2] == 0).all()
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.125)):
        check_attend(got, want, bound, f"plan {plan}")
