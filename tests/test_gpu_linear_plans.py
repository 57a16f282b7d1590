"""attn_linear's two forms under forced plans, chunks in several passes, and
what conv_causal, attn_linear and sample_logits refuse of their views."""
from __future__ import annotations

import numpy as np
import pytest

import qmr
from linear_cases import Conv, Linear, dispatch
from sample_cases import Sample
from test_gpu_linear import CHUNKS

pytestmark = pytest.mark.gpu


@pytest.fixture()
def planned(gpu):
    yield gpu.set_gemv_plan
    gpu.set_gemv_plan(0, 0)


KERNELS = {1: "attn_linear_tokens_kernel", 2: "linear_scan_kernel"}


@pytest.mark.parametrize("plan", [100, 200, 202, 204, 203])
@pytest.mark.parametrize("heads", [(2, 4, 64, 64), (1, 2, 128, 120), (1, 1, 256, 256), (1, 3, 8, 200)])
@pytest.mark.parametrize("delta", [True, False])
def test_forced_plans(gpu, planned, plan, heads, delta):
    planned(-8, plan)
    for counts in ([1], [3, 1, 2], [33, 0, 64], [150, 31]):
        case = Linear(counts, *heads, delta=delta, behind=2)
        case.check(gpu, CHUNKS, f"{plan} {counts}", pad=8)
        assert gpu.last_hip_kernel() == KERNELS[plan // 100]


@pytest.mark.parametrize("pad", [0, 1 << 22])
def test_both_forms_keep_the_same_rows(gpu, planned, pad):
    """Rows so far apart that a chunk's do not fit 32-bit offsets go token after
    token, also where chunks are asked for."""
    case = Linear([9, 40], 1, 2, 16, 16)
    case.check(gpu, CHUNKS, pad=pad)
    planned(-8, 200)
    got, after = case.check(gpu, CHUNKS, pad=pad)
    assert gpu.last_hip_kernel() == KERNELS[1 if pad else 2]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("counts", [[3000], [900, 1, 0, 1400, 32, 700], [64] * 40])
def test_chunks_in_passes_are_those_in_one(gpu, counts, delta):
    """The static scratch holds the chunks of some of these tokens alone; states
    go from one pass to the next, and no bit depends on it."""
    case = Linear(counts, 8, 16, 128, 128, delta=delta)
    assert not np.isnan(case.state).any()
    out, after = case.run(gpu)
    got, state = case.run(gpu, static=True)
    assert gpu.last_hip_kernel() == KERNELS[2]
    assert np.array_equal(out, got) and np.array_equal(after, state)
    if sum(counts) == 3000:
        small = Linear(counts, 1, 1, 128, 128, delta=delta)
        small.check(gpu, CHUNKS, static=True)


def test_the_largest_dimensions_through_the_scratch(gpu):
    # A chunk's operands take 64 KB a key head and 9 KB a value head. Four chunks
    # are 5.9 MB; eleven are more than the scratch, and so is a state of 256 KB
    # for each of 48 heads, twice, that passes would hand on.
    case = Linear([70, 3], 16, 48, 256, 256)
    case.check(gpu, CHUNKS, static=True)
    assert gpu.last_hip_kernel() == KERNELS[2]
    case = Linear([300, 3], 16, 48, 256, 256)
    case.check(gpu, CHUNKS, static=True)
    assert gpu.last_hip_kernel() == KERNELS[1]
    case = Linear([70, 3], 2, 4, 256, 256)
    case.check(gpu, CHUNKS, static=True)
    assert gpu.last_hip_kernel() == KERNELS[2]


@pytest.mark.parametrize("factor", [1e-30, 1e-12, 1e15, 1e30])
@pytest.mark.parametrize("n", [4, 100])
def test_states_and_values_of_any_size(gpu, factor, n):
    """Everything is linear in the state and the values together, and powers of
    two are exact: a factor of 2^k moves no bit but the exponent's."""
    two = 2.0 ** round(np.log2(factor))
    case = Linear([n], 1, 2, 64, 64, out_eps=0.0)
    out, after = case.run(gpu)
    case.v, case.state = (case.v * two).astype(np.float32), (case.state * two).astype(np.float32)
    got, state = case.run(gpu)
    if factor > 1e-20:
        assert np.array_equal(got, out * np.float32(two)) and np.array_equal(state, after * np.float32(two))
    else:  # products of terms go below FP32's normal numbers, each off by 2^-126 at most there
        assert np.abs(got / two - out).max() < 1e-4 * np.abs(out).max()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("length", [1.5, 40.0])
def test_long_keys(gpu, delta, length):
    """Keys longer than 1: with the delta rule a state can grow without bound;
    what comes is FP32 arithmetic's token after token, where that stays finite."""
    case = Linear([70, 9], 1, 2, 32, 32, qk_eps=0.0, out_eps=0.0, delta=delta, gates=False)
    case.k *= np.float32(length)
    case.a[:] = -3.0
    out, after = case.run(gpu)
    want, _, states, _ = case.want(1)
    with np.errstate(all="ignore"):
        fits = np.abs(want).max(1) < 1e30
        assert fits[:5].all()
        # A token takes on what the state was off by before it, length^2 times as much
        # at most: ten tokens of that are compared.
        for first in (0, 70):
            part = slice(first, first + 9)
            grown = np.cumprod(np.full(9, max(1.0, length ** 2 * 0.05) if delta else 1.0))[:, None]
            scale = np.maximum.accumulate(np.abs(want[part]).max(1))[:, None]
            assert (np.abs(out[part] - want[part]) <= 400 * 2.0 ** -24 * length ** 2 * grown * scale + 1e-30).all()


def views(gpu, name):
    """Buffers, offsets and words of a call that is taken, from one buffer each."""
    n = 4
    if name == "conv_causal":
        params = [1, n, 8, 4, 8, 8, 1, 1, 2, 1]
    elif name == "attn_linear":
        params = [1, n, 1, 2, 8, 8, 8, 8, 16, 2, 2, 16, 16, n, 1, 1, 0x3F000000, 0x358637BD, 0x358637BD, 2, 1]
    else:
        params = [n, 40, 40]
    sizes = qmr.dispatch_layout(name, params)[0]
    buffers = [gpu.alloc(s) for s in sizes]
    starts = {"conv_causal": 3, "attn_linear": 9}.get(name)
    if starts is not None:
        buffers[starts].write(np.array([0, n], np.uint32))
    return buffers, params, sizes


@pytest.mark.parametrize("name", ["conv_causal", "attn_linear", "sample_logits"])
def test_what_is_written_shares_no_byte_with_another_view(gpu, name):
    buffers, params, sizes = views(gpu, name)
    dispatch(gpu, name, buffers, params)
    for out in range({"conv_causal": 5, "attn_linear": 11, "sample_logits": 6}[name], len(buffers)):
        for other in range(len(buffers)):
            if other == out:
                continue
            shared = gpu.alloc(sizes[out] + sizes[other])
            for at_out, at_other in ((0, 0), (0, sizes[out] - 4), (sizes[other] - 4, 0)):
                mixed, offsets = list(buffers), [0] * len(buffers)
                mixed[out] = mixed[other] = shared
                offsets[out], offsets[other] = at_out, at_other
                with pytest.raises(qmr.QmrError, match="overlaps"):
                    dispatch(gpu, name, mixed, params, offsets)
            # One behind the other is well.
            if name != "sample_logits" and other in (3, 4, 9, 10):
                continue  # starts that are not there
            mixed, offsets = list(buffers), [0] * len(buffers)
            mixed[out] = mixed[other] = shared
            offsets[other] = sizes[out]
            dispatch(gpu, name, mixed, params, offsets)


def test_rows_beside_rows_of_one_buffer(gpu):
    case = Conv([3, 2], 8, 4)
    want, after = case.run(gpu)
    both = np.full((5, 20), 9.0, np.float32)
    both[:, :8] = case.x
    x, state = gpu.upload_f32(both), gpu.upload_f32(case.state)
    up = gpu.upload_bytes
    small = [up(case.w), up(case.b), up(case.starts), up(case.slots)]
    params = [2, 5, 8, 4, 20, 20, 1, 0, case.pool, 1]
    dispatch(gpu, "conv_causal", [x, *small, state, x], params, [0, 0, 0, 0, 0, 0, 32])
    got = x.read(np.float32, both.size).reshape(both.shape)
    assert np.array_equal(got[:, 8:16], want) and np.array_equal(got[:, :8], case.x) and (got[:, 16:] == 9).all()
    for offset in (0, 28, 52):  # in place, over its end, around the stride into the next row
        with pytest.raises(qmr.QmrError, match="overlaps"):
            dispatch(gpu, "conv_causal", [x, *small, state, x], [2, 4, 8, 4, 20, 20, 1, 0, case.pool, 1],
                     [0, 0, 0, 0, 0, 0, offset])


@pytest.mark.parametrize("name", ["conv_causal", "attn_linear", "sample_logits"])
def test_buffers_too_short_and_reference_mode(gpu, gpus, name):
    buffers, params, sizes = views(gpu, name)
    for i, size in enumerate(sizes):
        short = list(buffers)
        short[i] = gpu.alloc(size - 4) if size > 4 else None
        if short[i] is not None:
            with pytest.raises(qmr.QmrError):
                dispatch(gpu, name, short, params)
        with pytest.raises(qmr.QmrError):
            dispatch(gpu, name, buffers, params, [2 if j == i else 0 for j in range(len(sizes))])
    reference = gpus["reference"]
    other, params, _ = views(reference, name)
    with pytest.raises(qmr.QmrError, match="reference mode"):
        dispatch(reference, name, other, params)


def test_starts_that_are_no_ascent_stay_inside_the_rows(gpu):
    """Rows past the last, sequences that end before they begin or share rows:
    what comes is not defined, but other rows and slots stay as they were."""
    case = Linear([40, 3, 20], 1, 2, 32, 32, behind=9, pool=6, slots=[1, 2, 4])
    for starts in ([0, 72, 9, 0xFFFFFFFF], [50, 3, 2, 1], [0xFFFFFFFF, 0, 72, 30]):
        case.starts = np.array(starts, np.uint32)
        for counts in (8, 40):
            case.most = counts
            _, after = case.run(gpu, pad=3, shift=1)
            for slot in (0, 3, 5):
                assert np.array_equal(after[slot], case.state[slot])


def test_attention_and_draws_share_a_workspace(gpu):
    """One command: a long prompt, a draw, the same again; each as alone."""
    case, draw = Linear([500, 20], 2, 4, 64, 64), Sample(np.random.default_rng(3).standard_normal((5, 50001)), 1.0, 0, 0.9)
    other = qmr.Gpu("aligned")
    try:
        for static in (False, True):
            alone, drawn = case.run(gpu, static=static), draw.run(gpu, static=static)
            for _ in range(3):  # the first grows the workspace from nothing
                tokens, probs = draw.run(other, static=static)
                out, after = case.run(other, static=static)
                assert np.array_equal(out, alone[0]) and np.array_equal(after, alone[1])
                assert np.array_equal(tokens, drawn[0]) and np.array_equal(probs, drawn[1])
    finally:
        other.close()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("sizes", [(1e8, 1e8, 1e8), (1e20, 1.0, 1e-20), (1e-30, 1e10, 1e-30), (1.0, 1e36, 1.0),
                                   (0.0, 1e3, 1e-3), (1e-38, 0.0, 1e30)])
def test_values_far_larger_than_the_state(gpu, planned, sizes, delta):
    """From a state of zeros, values whose size changes from chunk to chunk and
    within one."""
    case = Linear([110, 40], 1, 2, 32, 32, out_eps=0.0, delta=delta)
    case.state[:] = 0
    for i, size in enumerate(sizes):
        case.v[37 * i:37 * (i + 1)] *= np.float32(size)
        case.v[110 + 13 * i:110 + 13 * (i + 1)] *= np.float32(size)
    for plan in (200, 100):
        planned(-8, plan)
        got, after = case.run(gpu)
        # R and U are two f16 terms, scaled to a largest of 2^5 to 2^6 in a column and
        # chunk: the second is off by 2^-25, so 2^-30 of that largest. Twice, over rows
        # of T at most 8 long.
        want, bound, states, state_bound = case.want(CHUNKS, 2.0 ** -30 * 2 * 8 if plan == 200 else 0.0)
        # Numbers below FP32's normal ones are off by its least step in each term.
        assert (np.abs(got - want) <= bound + 1e-36).all(), plan
        assert (np.abs(after - states) <= state_bound + 1e-36).all(), plan
