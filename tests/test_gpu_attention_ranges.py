"""attn_paged over key ranges of one block and more, and the ways they are joined."""
import numpy as np
import pytest

from attention_cases import Batch, attend, attend64, check_attend, from_half, make_pool, to_half

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]
# 16 rows a workgroup: as many ranges as there are blocks, ranges of two blocks
# or more, five and four (a join of a workgroup a row, and of a wave a row).
PLANS = [16511, 16040, 16020, 16005, 16004, 128009]


def run(gpu, kind, batch, heads, kv_heads, dim, plans=PLANS, **mask):
    rng = np.random.default_rng(dim + heads)
    q = rng.standard_normal((batch.tokens, heads, dim)).astype(np.float32)
    k, v = make_pool(batch, kv_heads, dim, kind, rng)
    scale = np.float32(dim ** -0.5)
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, np.float64(scale), **mask)
    try:
        for plan in plans:
            gpu.set_gemv_plan(-7, plan)
            got = attend(gpu, kind, q, k, v, batch, scale, **mask)
            check_attend(got, want, bound, f"plan {plan}: {kind} {heads}/{kv_heads}x{dim} {batch.new} {batch.lengths}")
            # Nothing is added up in an order that changes.
            assert np.array_equal(got, attend(gpu, kind, q, k, v, batch, scale, **mask), equal_nan=True)
    finally:
        gpu.set_gemv_plan(0, 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length", [31, 33, 95, 1001, 2079])
def test_single_tokens(gpu, kind, dim, length):
    run(gpu, kind, Batch([1, 1], [length, max(1, length // 3)], 32), 6, 1, dim)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 33, 64, 300])
def test_windows(gpu, kind, window):
    run(gpu, kind, Batch([1, 40, 3], [1400, 700, 64], 32), 7, 1, 64, window=window)
    run(gpu, kind, Batch([9], [701], 64), 3, 3, 128, window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_ragged(gpu, kind):
    run(gpu, kind, Batch([0, 2, 5, 33, 1], [10, 1, 3, 640, 900], 32, dropped=((3, 0), (3, 7), (4, 28))), 6, 2, 72)
    run(gpu, kind, Batch([3, 1], [500, 20], 64), 4, 2, 64, causal=False, max_keys=301)


@pytest.mark.parametrize("kind", KINDS)
def test_many_rows(gpu, kind):
    # 4200 rows: joined by a wave a row up to 16 ranges.
    run(gpu, kind, Batch([350], [700], 64), 12, 1, 64, plans=[16009, 16016, 16021])


@pytest.mark.parametrize("kind", KINDS)
def test_not_finite(gpu, kind):
    # Position 40 is an infinity in one value and a NaN in another: rows from
    # position 40 on are NaN there, the ones before are not.
    batch = Batch([30], [60], 32)
    infinity = to_half(np.float32([np.inf, np.nan]), kind)
    rng = np.random.default_rng(3)
    q = rng.standard_normal((30, 2, 64)).astype(np.float32)
    k, v = make_pool(batch, 1, 64, kind, rng)
    v[batch.table[0][1], 0, 8, [3, 60]] = infinity
    try:
        for plan in PLANS:
            gpu.set_gemv_plan(-7, plan)
            got = attend(gpu, kind, q, k, v, batch, 0.125)
            sees = np.arange(30, 60) >= 40
            assert not np.isfinite(got[sees][..., [3, 60]]).any() and np.isfinite(got[~sees]).all(), plan
            assert np.isfinite(np.delete(got, [3, 60], axis=2)).all(), plan
    finally:
        gpu.set_gemv_plan(0, 0)
