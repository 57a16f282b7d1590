"""attn_paged where one key has nearly all of a row's weight and a value of zero,
so that the row is what small weights make of the other values."""
import numpy as np
import pytest

from attention_cases import Batch, attend, from_half, make_pool, to_half

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]
# The planner's choice, and each kernel with and without key ranges.
PLANS = [0, 16001, 16003, 128001, 128003]


def scores_bound(largest: float, keys: int) -> float:
    """Relative to sum p|v|, where a score is one product. It is off by 4.5e-7
    of itself: the query's scaling and its place against the maximum round by
    6e-8 each (three times), its terms by 1.2e-7 and the sum of their products
    by as much; so p moves by that much of the largest score, and so does the
    maximum that it stands against. 2.4e-7 a block of 32 keys as a random walk.
    1e-6 for the exponential, the division and the weights' own 22 bits.
    """
    return 2 * 4.5e-7 * largest + 2.4e-7 * np.sqrt(keys / 32) + 1e-6


# An f16 weight is off by 2^-36 of its row's largest, which is no more than that of
# the sum of all, and so is what it makes of a value.
WEIGHT = {"bf16": 0.0, "f16": 2.0 ** -36}


def sink_case(kind, batch, heads, kv_heads, dim, gap, spread, seed):
    """Queries of one element, so that scores are the keys' first ones: `gap` for
    position 0, normal ones of `spread` for the others. Values are 0 and positive."""
    rng = np.random.default_rng(seed)
    k, v = make_pool(batch, kv_heads, dim, kind, rng)
    shape = k.shape
    k[...] = 0
    k[..., 0] = to_half(spread * rng.standard_normal(shape[:3]), kind)
    v[...] = to_half(rng.uniform(0.5, 1.5, shape), kind)
    for s in range(len(batch.new)):
        k[batch.table[s, 0], :, 0, 0] = to_half(np.float32([gap]), kind)[0]
        v[batch.table[s, 0], :, 0] = 0
    q = np.zeros((batch.tokens, heads, dim), np.float32)
    q[..., 0] = rng.uniform(0.99, 1.01, (batch.tokens, heads))
    return q, k, v


def check(gpu, kind, batch, heads, kv_heads, dim, gap, spread=0.5, plans=PLANS, seed=0):
    q, k, v = sink_case(kind, batch, heads, kv_heads, dim, gap, spread, seed)
    k64, v64 = from_half(k, kind), from_half(v, kind)
    group, page = heads // kv_heads, batch.page
    want, lost = np.zeros(q.shape), np.zeros(q.shape)
    for s, n in enumerate(batch.new):
        at = np.arange(batch.lengths[s])
        kk, vv = k64[batch.table[s, at // page], :, at % page, 0], v64[batch.table[s, at // page], :, at % page]
        for i in range(n):
            seen = batch.lengths[s] - n + i + 1
            for h in range(heads):
                t = int(batch.starts[s]) + i
                p = np.exp(kk[:seen, h // group] * float(q[t, h, 0]) - gap)
                want[t, h] = p @ vv[:seen, h // group] / p.sum()
                lost[t, h] = WEIGHT[kind] * vv[:seen, h // group].sum(axis=0)
    bound = scores_bound(1.01 * gap, max(batch.lengths))
    try:
        for plan in plans:
            gpu.set_gemv_plan(-7, plan)
            got = attend(gpu, kind, q, k, v, batch, 1.0)
            off = np.abs(got - want) / (bound * want + lost)
            assert off.max() <= 1, f"plan {plan}: {off.max():.2f} times the bound"
    finally:
        gpu.set_gemv_plan(0, 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gap", [8.0, 10.0, 12.0, 14.0])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_sinks(gpu, kind, gap, dim):
    check(gpu, kind, Batch([1], [4001], 64), 4, 2, dim, gap, seed=dim)
    check(gpu, kind, Batch([33, 2], [4096, 1500], 64), 2, 1, dim, gap, seed=dim)


@pytest.mark.parametrize("kind", KINDS)
def test_sink_over_a_long_history(gpu, kind):
    check(gpu, kind, Batch([1, 2], [32768, 20001], 128), 2, 1, 64, 10.0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gap", [14.0, 17.0, 22.0, 27.0])
@pytest.mark.parametrize("lengths", [(2, 3), (40, 70)])
def test_sinks_over_few_keys(gpu, kind, gap, lengths):
    # Weights that are all alike: what each of them loses does not average out.
    for spread in (0.0, 2.0):
        check(gpu, kind, Batch([1, 1], lengths, 32), 6, 2, 128, gap, spread)
        check(gpu, kind, Batch([1, 1], lengths, 32), 2, 2, 256, gap, spread)
        check(gpu, kind, Batch([1, 2], lengths, 32), 2, 2, 40, gap, spread)
