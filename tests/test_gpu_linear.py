"""attn_linear against its definition in 64 bits."""
import numpy as np
import pytest

from linear_cases import FRESH, Linear

pytestmark = pytest.mark.gpu

# Roundings of one token, relative to the lengths of what they act on: the
# norm of k (10 for its sum, root, quotient, product), a column's product with
# it (dk / 32 in sequence, 9 to join), the correction and the update (6).
# A chunk of 64 tokens instead solves for its corrections at once: products of
# dk and of 64 terms, summed by fours, one on the other (64 + 32 + 32), over an
# inverse whose rows are at most 8 long where a correction is 1.
TOKENS = 48
CHUNKS = 400

COUNTS = [[1], [2], [3, 0, 1], [1] * 6, [17], [64], [65, 1, 0, 63], [130, 5]]
DIMS = [(1, 1, 8, 8), (2, 4, 32, 32), (1, 3, 128, 128), (2, 2, 40, 24), (1, 2, 64, 136), (1, 1, 256, 256), (3, 3, 96, 80)]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("heads", DIMS)
@pytest.mark.parametrize("delta", [True, False])
def test_linear(gpu, counts, heads, delta):
    Linear(counts, *heads, delta=delta).check(gpu, CHUNKS if max(counts) > 3 else TOKENS)


@pytest.mark.parametrize("gates", [True, False])
@pytest.mark.parametrize("qk_eps", [0.0, 1e-6])
@pytest.mark.parametrize("out_eps", [0.0, 1e-5])
@pytest.mark.parametrize("counts", [[1, 2], [70, 33]])
def test_switches(gpu, gates, qk_eps, out_eps, counts):
    for delta in (True, False):
        Linear(counts, 2, 6, 64, 64, gates=gates, delta=delta, qk_eps=qk_eps, out_eps=out_eps).check(gpu, CHUNKS)


@pytest.mark.parametrize("pad,shift", [(0, 1), (3, 2), (4, 4), (13, 0)])
@pytest.mark.parametrize("counts", [[1, 1, 2], [66, 20]])
def test_strides_and_rows_behind(gpu, pad, shift, counts):
    Linear(counts, 2, 4, 48, 72, behind=5).check(gpu, CHUNKS, pad=pad, shift=shift)


@pytest.mark.parametrize("counts", [[2, 1], [100, 65]])
def test_one_row_of_decays_for_all_tokens(gpu, counts):
    Linear(counts, 2, 2, 32, 64, gates=False, delta=False, fixed=True, qk_eps=0.0).check(gpu, CHUNKS)


@pytest.mark.parametrize("n", [1, 3, 70])
def test_states_that_are_fresh_shared_or_not_there(gpu, n):
    # Slot 2 has two sequences: the first one has it. Slots 9 and up are past the pool.
    case = Linear([n, 2, n, 1, n], 1, 2, 32, 32, pool=6, slots=[2, 2 | FRESH, 5 | FRESH, 9, 0x7FFFFFFF])
    _, after = case.check(gpu, CHUNKS)
    for slot in (0, 1, 3, 4):
        assert np.array_equal(after[slot], case.state[slot])
    case.state[5] = np.nan
    out, after = case.run(gpu)
    assert np.isfinite(out).all() and np.isfinite(after[5]).all()
    Linear([2] * 130, 1, 1, 16, 8, pool=3, slots=[1] * 129 + [2]).check(gpu, CHUNKS)


@pytest.mark.parametrize("counts", [[1, 2], [90, 3]])
def test_states_are_kept_only_on_demand(gpu, counts):
    case = Linear(counts, 2, 4, 64, 64, keep=False)
    _, after = case.check(gpu, CHUNKS)
    assert np.array_equal(after, case.state)


@pytest.mark.parametrize("most", [1, 3, 64, 80])
def test_at_most_so_many_tokens_of_a_sequence(gpu, most):
    case = Linear([100, 2, 70], 1, 2, 32, 32, most=most)
    out, _ = case.run(gpu)
    want, bound, states, state_bound = case.want(CHUNKS)
    assert (np.abs(out - want) <= bound).all()  # rows behind them as they were


@pytest.mark.parametrize("delta", [True, False])
def test_parts_of_a_sequence_make_the_whole(gpu, delta):
    whole = Linear([200], 1, 2, 64, 64, delta=delta)
    want, bound, state, state_bound = whole.want(CHUNKS)
    first, at, got = whole.state, 0, []
    for n in (1, 70, 1, 3, 64, 61):
        case = Linear([n], 1, 2, 64, 64, delta=delta, slots=whole.slots, pool=whole.pool)
        rows = slice(at, at + n)
        for name in ("q", "k", "v", "a", "b", "z"):
            setattr(case, name, getattr(whole, name)[rows])
        case.a_log, case.dt_bias, case.norm, case.state = whole.a_log, whole.dt_bias, whole.norm, first
        out, first = case.run(gpu)
        got.append(out)
        at += n
    assert (np.abs(np.concatenate(got) - want) <= bound).all()
    assert (np.abs(first - state) <= state_bound).all()


@pytest.mark.parametrize("n", [2, 150])
@pytest.mark.parametrize("delta", [True, False])
def test_decays_at_their_ends(gpu, n, delta):
    # No decay at all, a state forgotten at once, and both in turn.
    case = Linear([n], 1, 4, 32, 32, gates=False, delta=delta)
    case.a[:, 0] = 0
    case.a[:, 1] = -np.inf
    case.a[:, 2] = -1e30
    case.a[:, 3] = np.where(np.arange(n) % 5 == 1, -np.inf, -0.01)
    case.check(gpu, CHUNKS)
    # Steps of the gates' formula that overflow, or are nothing.
    case = Linear([n], 1, 4, 32, 32, delta=delta)
    case.a[:, 0], case.a[:, 1], case.a[:, 2] = 1e4, -1e4, 88.0
    case.a_log[3] = -100
    case.check(gpu, CHUNKS)


def test_a_long_sequence(gpu):
    Linear([1500], 1, 2, 128, 128).check(gpu, CHUNKS)
    Linear([777, 1, 900], 1, 1, 64, 64, delta=False).check(gpu, CHUNKS)


@pytest.mark.parametrize("name,width", [("q", 0), ("k", 0), ("v", 0), ("a", 1), ("b", 1), ("z", 0)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_what_is_not_finite_reaches_no_earlier_token_and_no_other_sequence(gpu, name, width, value):
    case = Linear([90, 90], 1, 2, 32, 32, behind=6)
    want, bound, states, state_bound = case.want(CHUNKS)
    array = getattr(case, name)
    array[70, 0] = value
    array[180:] = np.nan
    out, after = case.run(gpu)
    clean = np.ones(out.shape, bool)
    clean[70:90] = False
    assert (np.abs(out - want)[clean] <= bound[clean]).all()
    second = case.slots[1]
    assert (np.abs(after[second] - states[second]) <= state_bound[second]).all()
    if name in ("k", "v"):
        assert not np.isfinite(out[70, 0])


def test_a_state_that_is_not_finite_stays_in_its_head(gpu):
    for n in (1, 80):
        case = Linear([n, n], 1, 2, 32, 32)
        want, bound, _, _ = case.want(CHUNKS)
        case.state[case.slots[0], 0] = np.nan
        out, after = case.run(gpu)
        assert np.isnan(out[:n, :32]).all()
        assert (np.abs(out - want)[:n, 32:] <= bound[:n, 32:]).all()
        assert (np.abs(out - want)[n:] <= bound[n:]).all()


@pytest.mark.parametrize("counts", [[1, 1, 3], [300, 2, 65]])
def test_static_entry(gpu, counts):
    case = Linear(counts, 2, 4, 64, 64)
    out, after = case.run(gpu)
    got, state = case.run(gpu, static=True)
    assert np.array_equal(out, got) and np.array_equal(after, state)
