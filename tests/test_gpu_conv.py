"""conv_causal against its definition in 64 bits."""
import numpy as np
import pytest

from linear_cases import FRESH, Conv

pytestmark = pytest.mark.gpu

COUNTS = [[1], [2], [3], [4], [37], [1] * 5, [3, 0, 1, 9], [0, 70, 2], [33, 64, 1]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("channels,width", [(8, 4), (1, 3), (260, 4), (1001, 2), (30, 4)])
def test_conv(gpu, counts, channels, width):
    Conv(counts, channels, width).check(gpu)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("pad,shift", [(0, 1), (3, 2), (5, 0), (4, 4)])
def test_strides_and_switches(gpu, silu, bias, pad, shift):
    for channels in (12, 7):
        Conv([5, 41], channels, 4, silu=silu, bias=bias, behind=3).check(gpu, pad=pad, shift=shift)


def test_long_sequence_and_many(gpu):
    Conv([2500], 64, 4).check(gpu)
    Conv([1 + i % 3 for i in range(150)], 16, 3, behind=2).check(gpu)


def test_states_that_are_fresh_shared_or_not_there(gpu):
    # Slot 2 has two sequences: the first one has it. Slots 9 and up are past the pool.
    c = Conv([4, 2, 3, 1, 2], 12, 4, pool=6, slots=[2, 2 | FRESH, 5 | FRESH, 9, 0x7FFFFFFF])
    _, after = c.check(gpu)
    for slot in (0, 1, 3, 4):
        assert np.array_equal(after[slot], c.state[slot])
    # A fresh state is not read.
    c.state[5] = np.nan
    y, after = c.run(gpu)
    assert np.isfinite(y).all() and np.isfinite(after[5]).all()
    # One slot for more sequences than a wave has lanes.
    Conv([2] * 130, 8, 4, pool=3, slots=[1] * 129 + [2]).check(gpu)


@pytest.mark.parametrize("counts", [[1, 2, 9], [40]])
def test_states_are_kept_only_on_demand(gpu, counts):
    c = Conv(counts, 20, 4, keep=False)
    _, after = c.check(gpu)
    assert np.array_equal(after, c.state)


def test_parts_of_a_sequence_make_the_whole(gpu):
    whole = Conv([57], 24, 4, bias=True)
    want, state = whole.run(gpu)
    got, at = [], 0
    for n in (1, 1, 2, 30, 3, 20):
        c = Conv([n], 24, 4, bias=True, slots=whole.slots, pool=whole.pool)
        c.x, c.w, c.b, c.state = whole.x[at:at + n], whole.w, whole.b, whole.state
        y, whole.state = c.run(gpu)
        got.append(y)
        at += n
    assert np.array_equal(np.concatenate(got), want) and np.array_equal(whole.state, state)


def test_what_is_not_finite_stays_in_its_window(gpu):
    c = Conv([20, 20], 8, 4, behind=4, slots=[0, 1])
    c.x[7, 3], c.x[25, 2], c.x[40:] = np.nan, np.inf, np.nan
    y, after = c.run(gpu)
    bad = ~np.isfinite(y)
    assert bad[7:11, 3].all() and bad.sum() == bad[7:11, 3].sum() + bad[25:29, 2].sum()
    assert np.isfinite(after).all()
    assert (y[40:] == 9).all()
