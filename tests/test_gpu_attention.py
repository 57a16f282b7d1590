"""attn_paged_bf16 / attn_paged_f16 against the definition in 64 bits."""
import numpy as np
import pytest

import qmr
from attention_cases import Batch, attend, attend64, check_attend, from_half, make_pool, to_half

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]
# The planner's choice, and each kernel with and without key ranges.
PLANS = [0, 16001, 16003, 128001, 128002]


def under_plans(gpu, call):
    """(plan, call()) under each plan, the planner's last."""
    try:
        for plan in PLANS[1:]:
            gpu.set_gemv_plan(-7, plan)
            yield plan, call()
    finally:
        gpu.set_gemv_plan(0, 0)
    yield 0, call()



def run(gpu, kind, batch, heads, kv_heads, dim, seed=0, spread=1.0, **how):
    rng = np.random.default_rng(seed)
    q = (spread * rng.standard_normal((batch.tokens, heads, dim))).astype(np.float32)
    k, v = make_pool(batch, kv_heads, dim, kind, rng)
    scale = how.pop("scale", dim ** -0.5)
    mask = {n: how[n] for n in ("causal", "window", "max_keys") if n in how}
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, np.float32(scale).astype(np.float64), **mask)
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, scale, **how)):
        check_attend(got, want, bound, f"plan {plan}: {kind} {heads}/{kv_heads}x{dim} {batch.new} {batch.lengths}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 72, 128, 136, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2)])
def test_head_sizes(gpu, kind, dim, heads, kv_heads):
    run(gpu, kind, Batch([1, 3, 5], [1, 37, 200], 32), heads, kv_heads, dim, seed=dim)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(24, 4), (14, 2), (40, 2), (5, 5), (33, 1)])
def test_head_groups(gpu, kind, heads, kv_heads):
    run(gpu, kind, Batch([1, 2, 4, 1], [65, 64, 96, 500], 64), heads, kv_heads, 64, seed=heads)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 1000, 4097])
@pytest.mark.parametrize("page", [32, 128])
def test_one_token(gpu, kind, length, page):
    run(gpu, kind, Batch([1], [length], page), 12, 2, 128, seed=length)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,new,length", [(64, 17, 17), (64, 130, 131), (128, 100, 333), (128, 257, 257),
                                            (256, 65, 400), (256, 129, 129), (72, 97, 500)])
def test_chunks(gpu, kind, dim, new, length):
    run(gpu, kind, Batch([new], [length], 64), 6, 2, dim, seed=new)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
def test_windows(gpu, kind, window):
    run(gpu, kind, Batch([1, 70, 3], [400, 200, 64], 32), 4, 2, 64, seed=window, window=window)
    run(gpu, kind, Batch([1, 9], [1400, 1300], 32), 4, 1, 128, seed=window, window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_all_keys(gpu, kind):
    run(gpu, kind, Batch([40, 1, 7], [90, 33, 7], 32), 4, 2, 64, causal=False)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_keys(gpu, kind):
    # No new tokens; no cache; fewer positions than new tokens (the first ones
    # have no key); rows of a sequence whose only pages are past the pool.
    run(gpu, kind, Batch([0, 2, 5, 3, 0], [10, 0, 3, 40, 0], 32, dropped=((3, 0), (3, 1))), 6, 2, 64)
    rng = np.random.default_rng(1)
    batch = Batch([2], [0], 32)
    k, v = make_pool(batch, 1, 64, kind, rng)
    assert (attend(gpu, kind, np.ones((2, 2, 64), np.float32), k, v, batch, 0.1) == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_past_the_pool_hold_nothing(gpu, kind):
    run(gpu, kind, Batch([1, 40], [300, 299], 32, dropped=((0, 0), (0, 4), (1, 3), (1, 8))), 6, 2, 128)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("column", [0, 1, 2, 3, 4])
def test_dropped_pages_behind_garbage(gpu, kind, column):
    # The last block's free slots hold NaN or infinities; a page that is not
    # there comes after it, whichever block that is.
    run(gpu, kind, Batch([3], [5 * 32 + 3], 32, dropped=((0, column),)), 2, 1, 64)
    run(gpu, kind, Batch([3], [5 * 32 + 3], 32, dropped=((0, column), (0, (column + 1) % 5))), 2, 1, 256)


@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences(gpu, kind):
    # More than a wave's 64, with empty ones among them.
    rng = np.random.default_rng(3)
    new = [int(n) for n in rng.integers(0, 4, 150)]
    lengths = [n + int(o) for n, o in zip(new, rng.integers(0, 120, 150))]
    run(gpu, kind, Batch(new, lengths, 32), 4, 2, 64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,shift", [(0, 1), (3, 0), (8, 4), (5, 2)])
def test_strides_and_offsets(gpu, kind, pad, shift):
    run(gpu, kind, Batch([3, 50], [90, 77], 32), 6, 2, 72, pad=pad, shift=shift)
    run(gpu, kind, Batch([1, 1], [900, 77], 32), 6, 2, 128, pad=pad, shift=shift)


@pytest.mark.parametrize("kind", KINDS)
def test_max_keys(gpu, kind):
    run(gpu, kind, Batch([1, 5], [300, 90], 32), 4, 2, 64, max_keys=77)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("spread,scale", [(1.0, 1.0), (1e-4, 0.1), (3e4, 1e-5), (1e-30, 0.1), (0.0, 1.0), (1e30, 1e-31)])
def test_query_ranges(gpu, kind, spread, scale):
    # Peaked rows, queries beyond and below the 16-bit range, zero queries.
    run(gpu, kind, Batch([2, 33], [400, 100], 32), 4, 2, 128, spread=spread, scale=scale)


@pytest.mark.parametrize("kind", KINDS)
def test_rising_scores(gpu, kind):
    # Every block's scores exceed the ones before: the running maximum moves
    # each time, by less and by more than it may lag.
    batch = Batch([1, 40], [700, 640], 32)
    rng = np.random.default_rng(5)
    k, v = make_pool(batch, 1, 64, kind, rng)
    q = np.ones((batch.tokens, 2, 64), np.float32)
    for s, length in enumerate(batch.lengths):
        for j in range(length):
            k[batch.table[s, j // 32], 0, j % 32] = to_half(np.full(64, (j // 32) * (0.05 if j % 2 else 0.4)), kind)
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, float(np.float32(0.3)))
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.3)):
        check_attend(got, want, bound, f"plan {plan}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [4, 40])
def test_hidden_values_do_not_reach_rows(gpu, kind, new):
    # A NaN and an infinity in keys and values that only later tokens see, and
    # in values that a window has left behind.
    batch = Batch([new], [100 + new], 32)
    rng = np.random.default_rng(6)
    k, v = make_pool(batch, 1, 64, kind, rng)
    q = rng.standard_normal((new, 4, 64)).astype(np.float32)
    nan, inf = to_half(np.array([np.nan, np.inf], np.float32), kind)
    at = 100 + new - 1  # the last token's own position
    for pos, bits in ((at, nan), (12, inf)):  # the first two tokens still see position 12
        v[batch.table[0, pos // 32], 0, pos % 32, 5] = bits
        k[batch.table[0, pos // 32], 0, pos % 32, 7] = bits
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, 0.125, window=90)
    assert np.isfinite(want[2:-1]).all()
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.125, window=90)):
        check_attend(got[2:-1], want[2:-1], bound[2:-1], f"plan {plan}")
        for i in (0, 1, -1):
            assert not np.isfinite(want[i]).all() and not np.isfinite(got[i]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_every_row_sees_a_value_that_is_not_finite(gpu, kind):
    batch = Batch([5], [200], 32)
    rng = np.random.default_rng(16)
    k, v = make_pool(batch, 1, 64, kind, rng)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    v[batch.table[0, 2], 0, 9, 11] = to_half(np.array([np.nan], np.float32), kind)[0]
    want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, 0.125)
    for plan, got in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.125)):
        check_attend(got, want, bound, f"plan {plan}")


@pytest.mark.parametrize("kind", KINDS)
def test_rows_repeat(gpu, kind):
    # The same bits whatever else ran, and from the static scratch.
    rng = np.random.default_rng(8)
    for batch, heads, kv in ((Batch([1], [3000], 64), 12, 2), (Batch([37, 1], [300, 900], 64), 6, 2)):
        q = rng.standard_normal((batch.tokens, heads, 128)).astype(np.float32)
        k, v = make_pool(batch, kv, 128, kind, rng)
        for plan, first in under_plans(gpu, lambda: attend(gpu, kind, q, k, v, batch, 0.09)):
            gpu.set_gemv_plan(-7, plan)
            assert np.array_equal(first, attend(gpu, kind, q, k, v, batch, 0.09)), plan
        want, bound = attend64(q, from_half(k, kind), from_half(v, kind), batch, float(np.float32(0.09)))
        check_attend(attend(gpu, kind, q, k, v, batch, 0.09, static=True), want, bound)


def test_pools_past_32_bits(gpu):
    # A page whose keys start past 2^32 bytes, and past 2^32 halves.
    page, dim, kv = 1024, 256, 8
    pages = (2 ** 32) // (page * dim * kv) + 3
    rng = np.random.default_rng(9)
    kind = "f16"
    batch = Batch([1], [700], page, spare=0)
    batch.pages = pages
    k, v = (to_half(rng.standard_normal((1, kv, page, dim)), kind) for _ in range(2))
    q = rng.standard_normal((1, kv, dim)).astype(np.float32)
    kc, vc = (gpu.alloc(2 * pages * page * dim * kv) for _ in range(2))
    y = gpu.alloc_f32(kv * dim)
    for at in (pages // 2 + 2, pages - 1):
        batch.table[0, 0] = at
        kc.write(pack(k, "k"), offset=2 * at * page * dim * kv)
        vc.write(pack(v, "v"), offset=2 * at * page * dim * kv)
        params = [1, 1, kv, kv, dim, kv * dim, kv * dim, page, pages, 1, page, 1, 0, _word(0.0625)]
        gpu.dispatch("attn_paged_f16", [gpu.upload_f32(q), *batch.upload(gpu), kc, vc, y], params, group_size=64)
        one = Batch([1], [700], page, spare=0)
        want, bound = attend64(q, from_half(k, kind), from_half(v, kind), one, 0.0625)
        check_attend(gpu.read_f32(y, kv * dim).reshape(1, kv, dim), want, bound, f"page {at}")


def pack(x, which):
    from attention_cases import pack_k, pack_v

    return pack_k(x) if which == "k" else pack_v(x)


def _word(v):
    from attention_cases import f32_word

    return f32_word(v)


def test_refusals(gpu):
    batch = Batch([2], [40], 32)
    q = gpu.alloc_f32(4096)
    cache = gpu.alloc(2 * batch.pages * 2 * 32 * 64 + 64)
    base = [1, 2, 4, 2, 64, 256, 256, 32, batch.pages, batch.columns, 64, 1, 0, _word(0.1)]
    bufs = [q, *batch.upload(gpu), cache, gpu.alloc(2 * batch.pages * 2 * 32 * 64), gpu.alloc_f32(512)]

    def refused(match, buffers=bufs, offsets=None, params=base, name="attn_paged_f16"):
        with pytest.raises(qmr.QmrError, match=match):
            gpu.dispatch(name, buffers, params, offsets=offsets, group_size=64)

    refused("16-byte aligned", offsets=[0, 0, 0, 0, 4, 0, 0])
    refused("overlaps input buffer 0", buffers=[q, *bufs[1:6], q])
    refused("overlaps input buffer 4", buffers=[*bufs[:6], cache])
    refused("belongs|ends at", buffers=[*bufs[:6], gpu.alloc_f32(8)])
    refused("expected 7 buffers", buffers=bufs[:6])
    # Rows beside the queries in one buffer are no overlap.
    wide = [*base[:5], 512, 512, *base[7:]]
    gpu.dispatch("attn_paged_f16", [q, *bufs[1:6], q], wide, offsets=[0, 0, 0, 0, 0, 0, 1024], group_size=64)
    refused("overlaps", buffers=[q, *bufs[1:6], q], offsets=[0, 0, 0, 0, 0, 0, 1020], params=wide)
    with qmr.Gpu("aligned", reference=True) as ref:
        own = [ref.alloc(len(b)) for b in bufs]
        with pytest.raises(qmr.QmrError, match="reference mode"):
            ref.dispatch("attn_paged_f16", own, base, group_size=64)
