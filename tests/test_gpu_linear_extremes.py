"""attn_linear's chunks where sizes within one differ by many powers of two."""
import numpy as np
import pytest

from linear_cases import Linear

pytestmark = pytest.mark.gpu

# Roundings of one token at dk = 32, relative to the lengths of what they act
# on. A product of two-term operands is off by 6 (2^-23 each, and as much for the
# product left out) and adds up as many terms as its depth. S^T q, S^T k and M
# have dk of them, T R and M U 32, T's own rows 32 twice, gates and norms 40:
# 3 (6 + 32) + 2 (6 + 32) + 64 + 40.
ROUNDINGS = 294
# What is below FP32's normal numbers is off by its least step in each term.
LEAST = 1e-36


def plain(counts, delta, dv=32, **how):
    """A case without norms, of keys at most about 1 long."""
    return Linear(counts, 1, 2, 32, dv, gates=False, delta=delta, qk_eps=0.0, out_eps=0.0, **how)


def right(got, want, bound):
    assert np.isfinite(got).all()
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= bound + LEAST).all(), float((off / (bound + LEAST)).max())


def check(gpu, case):
    out, after = case.run(gpu)
    want, bound, states, state_bound = case.want(ROUNDINGS)
    right(out, want, bound)
    right(after, states, state_bound)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("size", [1e8, 1e10, 1e20])
@pytest.mark.parametrize("counts", [[32], [64], [20, 33]])
def test_large_values_of_zero_keys_beside_a_state_that_decays(gpu, delta, size, counts):
    """Keys of zero take nothing on, whatever their values: the state is what
    its decays leave, e^-70 of it."""
    case = plain(counts, delta)
    for first, n in zip(case.starts, counts):
        rows = slice(int(first), int(first) + min(n, 32))
        case.k[rows] = 0
        case.v[rows] *= np.float32(size)
        case.a[rows] = -70.0 / min(n, 32)
    check(gpu, case)


@pytest.mark.parametrize("size", [200.0, 5000.0, 1e9, 1e18])
@pytest.mark.parametrize("zeros", [0, 256, 300])
def test_long_keys_behind_values_of_zero(gpu, size, zeros):
    """Columns whose values and states are zero for some chunks, then of size 1
    to 60, along keys that are long: sums stay far from FP32's largest number."""
    case = plain([400], False)
    rng = np.random.default_rng(zeros)
    case.k *= np.float32(size)
    case.v[:] = rng.choice([-1, 1], case.v.shape) * rng.uniform(1, 60, case.v.shape)
    case.v[:zeros, ::2] = 0
    case.state[..., ::2] = 0
    if size == 1e18:
        case.v *= np.float32(1e16)
    check(gpu, case)


def test_columns_of_zeros_keep_their_room(gpu):
    """Nine chunks of values of zero, from a state of zeros, leave a column as it
    was: what follows has the bits that it has alone."""
    for delta in (True, False):
        both = plain([288 + 70], delta, slots=[0], pool=1)
        both.state[:] = 0
        both.v[:288] = 0
        both.v[288:] *= np.float32(1000)
        alone = plain([70], delta, slots=[0], pool=1)
        for name in ("q", "k", "v", "a", "b", "z"):
            setattr(alone, name, getattr(both, name)[288:])
        alone.state = both.state
        out, after = both.run(gpu)
        want, state = alone.run(gpu)
        assert np.array_equal(out[288:], want) and np.array_equal(after, state)
        assert not out[:288].any()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 20, 2.0 ** 30])
def test_a_long_key_takes_nothing_from_tokens_before_it(gpu, delta, size):
    case = plain([32, 61], delta)
    case.state[:] = 0
    case.k[31] *= np.float32(size)
    case.k[32 + 60] *= np.float32(size)
    out, _ = case.run(gpu)
    want, bound, _, _ = case.want(ROUNDINGS)
    before = np.ones(93, bool)
    before[[31, 92]] = False
    right(out[before], want[before], bound[before])


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 20, 2.0 ** 30])
def test_a_long_key_that_is_forgotten_takes_nothing_from_tokens_behind(gpu, size):
    case = plain([32, 61], False)
    for at in (3, 32 + 40):
        case.k[at] *= np.float32(size)
        case.a[at + 1] = -40.0
    check(gpu, case)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("size", [1e18, 1e35])
def test_a_key_past_all_bounds_reaches_no_token_before_it(gpu, delta, size):
    """Its own direction is no other key's, so that nothing but the state, along
    it, grows; what it leaves behind it may be infinite."""
    case = plain([32, 40], delta)
    case.k[:, 7] = 0
    for at in (31, 32 + 20):
        case.k[at] = 0
        case.k[at, 7] = size
    out, _ = case.run(gpu)
    want, bound, _, _ = case.want(ROUNDINGS)
    before = np.r_[0:31, 32:52]
    right(out[before], want[before], bound[before])


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("counts", [[1], [40], [300]])
def test_an_element_of_a_state_that_is_not_finite_stays_alone(gpu, value, counts):
    """Without the delta rule no element of a state meets another: outputs of its
    column are not finite, the rest of it is what it would be."""
    case = plain(counts, False, slots=[0], pool=1)
    want, bound, states, state_bound = case.want(ROUNDINGS)
    case.state[0, 1, 3, 5] = value
    out, after = case.run(gpu)
    other = np.ones(out.shape[1], bool)
    other[32 + 5] = False
    right(out[:, other], want[:, other], bound[:, other])
    assert not np.isfinite(out[:, 32 + 5]).any()
    assert not np.isfinite(after[0, 1, 3, 5])
    after[0, 1, 3, 5] = states[0, 1, 3, 5]
    right(after, states, state_bound)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [4, 100])
def test_states_near_the_largest_number(gpu, delta, n):
    """Sums of scaled rows stay below it where results do. (Columns this large have
    the least scale there is, so that bits may differ from a smaller one's.)"""
    case = plain([n], delta)
    case.v /= np.float32(8)
    case.state /= np.float32(8)
    out, after = case.run(gpu)
    assert max(np.abs(out).max(), np.abs(after).max()) < 2
    two = np.float32(2.0 ** 126)
    case.v, case.state = case.v * two, case.state * two
    check(gpu, case)


@pytest.mark.parametrize("length", [1.5, 40.0, 3e5])
def test_long_keys_without_the_delta_rule(gpu, length):
    """Every token and the states: nothing grows but by the keys' lengths."""
    case = plain([70, 9, 200], False)
    case.k *= np.float32(length)
    check(gpu, case)


@pytest.mark.parametrize("most", [1, 9, 32, 64, 80])
@pytest.mark.parametrize("delta", [True, False])
def test_states_of_the_first_tokens_of_a_sequence(gpu, most, delta):
    check(gpu, plain([100, 2, 70, 33], delta, most=most))
