"""sample_logits against its definition in 64 bits."""
import numpy as np
import pytest

from sample_cases import NONE, Sample, distribution

pytestmark = pytest.mark.gpu

INF = np.inf


def logits(rows, vocab, seed=0, spread=2.5):
    rng = np.random.default_rng(seed + vocab)
    x = spread * rng.standard_normal((rows, vocab))
    for r in range(rows):
        at = rng.integers(0, vocab, min(40, vocab))
        x[r, at] += 12 * rng.random(len(at))
    return x.astype(np.float32)


SETTINGS = [  # temperature, k, p, min_p
    (1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (0.7, 0, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 50, 0.9, 0.02),
    (0.0, 0, 1.0, 0.0), (2.0, 1, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (0.05, 0, 0.999, 0.0), (30.0, 0, 0.6, 0.0),
    (1.0, 1000, 0.99999, 1e-6), (5.0, 0, 1.0, 1.0),
]


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4097, 32001])
@pytest.mark.parametrize("setting", SETTINGS)
def test_sample(gpu, vocab, setting):
    Sample(logits(9, vocab), *setting).check(gpu)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_a_whole_vocabulary(gpu, rows):
    some = [SETTINGS[i % len(SETTINGS)] for i in range(rows + 1)][1:]
    Sample(logits(rows, 248320), *zip(*some)).check(gpu)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 3), (4, 4)])
def test_strides(gpu, pad, shift):
    for vocab in (1001, 4096):
        Sample(logits(5, vocab), *zip(*SETTINGS[:5])).check(gpu, pad=pad, shift=shift)


def test_many_rows(gpu):
    n = 700
    some = [SETTINGS[i % len(SETTINGS)] for i in range(n)]
    Sample(logits(n, 333), *zip(*some)).check(gpu)


@pytest.mark.parametrize("vocab", [5, 1500, 70001])
def test_ties_go_to_the_lowest_index(gpu, vocab):
    x = np.zeros((4, vocab), np.float32)
    x[1, vocab // 2:] = 3
    x[2] = np.arange(vocab) % 3
    x[3] = -0.0
    x[3, ::2] = 0.0
    for setting in SETTINGS:
        Sample(x, *setting, u=[0.0, 0.3, 0.7, 0.999999]).check(gpu)
    tokens, _ = Sample(x, 0.0).run(gpu)
    assert list(tokens) == [0, vocab // 2, 2, 0]
    # Three of the ties are kept.
    tokens, probs = Sample(x, 1.0, k=3, u=0.99).check(gpu)
    assert tokens[0] == 2 and abs(probs[0] - 1 / 3) < 1e-7


@pytest.mark.parametrize("setting", SETTINGS)
def test_masks_and_what_is_not_finite(gpu, setting):
    x = logits(8, 3000)
    x[0] = -INF
    x[1] = np.nan
    x[2, 5:] = -INF
    x[3, ::2] = np.nan
    x[4, 100] = x[4, 2000] = INF
    x[5, 10:] = np.finfo(np.float32).min
    x[6] = -INF
    x[6, 2999] = np.finfo(np.float32).min
    x[7, :] = np.finfo(np.float32).max
    x[7, 3] = np.finfo(np.float32).min
    tokens, probs = Sample(x, *setting).check(gpu)
    assert tokens[0] == tokens[1] == NONE and tokens[6] == 2999 and tokens[2] < 5 and tokens[3] % 2 == 1
    assert tokens[4] in (100, 2000) and probs[6] == 1


def test_settings_at_their_ends(gpu):
    x = logits(1, 2000).repeat(9, axis=0)
    s = Sample(x, temperature=[np.nan, -1, np.inf, 1e-38, 1, 1, 1, 1, 1], k=[0, 0, 0, 0, 2000, 4000, NONE, 0, 0],
               p=[1, 1, 1, 1, 1, 1, 1, np.nan, -1], min_p=[0, 0, 0, 0, np.nan, -1, 2, 0, 0], u=0.5)
    s.check(gpu)
    for u in (-1.0, 0.0, 1.0, 2.0, np.nan, np.nextafter(np.float32(1), np.float32(0))):
        Sample(x[:2], 0.9, p=[1.0, 0.5], u=u).check(gpu)


def test_drawn_tokens_follow_the_distribution(gpu):
    row = logits(1, 400, spread=1.0)
    n = 4000
    s = Sample(np.repeat(row, n, axis=0), 1.5, k=30, p=0.9, u=(np.arange(n) + 0.5) / n)
    tokens, _ = s.run(gpu)
    kept, share = distribution(row[0], np.float32(1.5), 30, np.float32(0.9), 0.0)
    # Evenly spread numbers meet a token's share to within one of them at either end.
    count = np.bincount(tokens, minlength=400)
    assert count.sum() == count[kept].sum() and (np.abs(count[kept] - n * share) <= 1.001).all()


def test_static_entry(gpu):
    s = Sample(logits(12, 32001), *zip(*SETTINGS))
    a, b = s.run(gpu), s.run(gpu, static=True)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("setting", [dict(k=50, p=0.9), dict(p=0.7), dict(min_p=0.02), dict(), dict(temperature=0.0)])
def test_the_largest_vocabulary(gpu, setting):
    """2^24 logits: weights are whole numbers of 2^-38 of the greatest, off by
    half of one each."""
    case = Sample(2 * np.random.default_rng(1).standard_normal((2, 1 << 24), np.float32), **{"temperature": 0.8, **setting})
    tokens, probs = case.run(gpu)
    for r, row in enumerate(case.logits):
        kept, share = distribution(row, case.temperature[r], case.k[r], case.p[r], case.min_p[r])
        # Off by 2^-39 each, of the greatest one's share; borders by as much.
        slip = len(kept) * 2.0 ** -39 * share.max() + 2.0 ** -30
        at = np.searchsorted(kept, tokens[r])
        assert kept[at] == tokens[r]
        up_to = np.cumsum(share)
        assert up_to[at] - share[at] - slip <= case.u[r] <= up_to[at] + slip, r
        # An FP32 number is off by up to 2^-24 of itself: 0.13468765 by 3.6e-9.
        assert abs(probs[r] - share[at]) <= slip + 2.0 ** -24 * share[at]


@pytest.mark.parametrize("live", [1, 2, 40, 63, 64, 65, 66, 130])
@pytest.mark.parametrize("setting", [dict(k=1), dict(k=64), dict(k=65), dict(p=0.5), dict(p=0.999), dict(min_p=0.3), dict(),
                                     dict(k=30, p=0.9, min_p=0.01)])
def test_few_tokens_stand_out(gpu, live, setting):
    """Some tokens above a floor that weighs next to nothing, many of them alike,
    and numbers at both ends and between."""
    rng = np.random.default_rng(live)
    rows = rng.standard_normal((12, 20000)).astype(np.float32) - 60
    for r, row in enumerate(rows):
        at = rng.permutation(20000)[:live]
        row[at] = rng.choice([0.0, 1.0, 1.5], live) if r % 2 else rng.uniform(-3, 3, live)
    case = Sample(rows, **setting, u=[0, 1, 0.5, *rng.random(9)])
    case.check(gpu)


def test_more_rows_than_the_workspace_holds(gpu):
    """Rows of 9000 take 84 KB each: 900 go in two turns, through the scratch in
    ten."""
    rng = np.random.default_rng(8)
    case = Sample(2 * rng.standard_normal((900, 9000)), rng.choice([0.0, 0.7, 1.2], 900), k=rng.choice([0, 1, 40], 900),
                  p=rng.choice([0.5, 0.9, 1.0], 900), min_p=rng.choice([0.0, 0.1], 900))
    tokens, probs = case.check(gpu)
    got, shares = case.run(gpu, static=True)
    assert np.array_equal(tokens, got) and np.array_equal(probs, shares)
