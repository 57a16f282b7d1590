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


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("element", [1.0, -1.0, 0.3, -0.3])
@pytest.mark.parametrize("infinity", [np.inf, -np.inf])
def test_keys_that_are_not_finite(gpu, kind, element, infinity):
    # Rows that see the key are NaN or infinite, be the score it gives plus or
    # minus infinity, and whether the query's element has 16 bits or more; rows
    # that do not are as without it.
    batch = Batch([40, 1, 1], [130, 300, 1], 32)
    q, k, v = inputs(kind, batch, 4, 2, 64, 4)
    q[..., 7] = element
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, 0.125)
    bits = to_half(np.float32([infinity]), kind)[0]
    for s, pos in ((0, 110), (1, 45), (2, 0)):
        k[batch.table[s, pos // 32], 0, pos % 32, 7] = bits
    sees = np.zeros((42, 4), bool)  # key-value head 0 is that of query heads 0 and 1
    sees[20:, :2] = True
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.125)):
        assert not np.isfinite(got[sees]).any(), plan
        check_attend(got[~sees], want[~sees], bound[~sees], f"plan {plan}")


@pytest.mark.parametrize("new", [3, 60])
def test_scores_below_fp32_have_no_weight(gpu, new):
    # A finite key of bf16 whose product with the query is past FP32's range.
    batch = Batch([new], [200], 32)
    q, k, v = inputs("bf16", batch, 2, 1, 64, 5)
    q[..., 7] = 10.0
    row = (batch.table[0, 1], 0, 8, 7)
    k[row] = 0
    _, bound = attend64(q, from_half(k, "bf16"), from_half(v, "bf16"), batch, 0.125)
    k[row] = to_half(np.float32([-1000.0]), "bf16")[0]
    want, _ = attend64(q, from_half(k, "bf16"), from_half(v, "bf16"), batch, 0.125)
    k[row] = to_half(np.float32([-3e38]), "bf16")[0]
    for plan, got in under_plans(gpu, lambda: attend(gpu, "bf16", q, k, v, batch, 0.125)):
        check_attend(got, want, bound, f"plan {plan}")
