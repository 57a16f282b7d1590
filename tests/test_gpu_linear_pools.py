"""States, rows and logits whose offsets pass 2^32 bytes."""
from __future__ import annotations

import numpy as np
import pytest

import qmr
from linear_cases import PAD, Conv, Linear, dispatch
from sample_cases import distribution
from test_gpu_linear import CHUNKS

pytestmark = pytest.mark.gpu


def far_state(gpu, per_slot: int, state: np.ndarray, slots, pool: int):
    """A pool of `pool` slots that holds `state`'s rows in those of `slots`."""
    assert pool * per_slot > 1 << 32
    buffer = gpu.alloc(pool * per_slot)
    for at, slot in enumerate(slots):
        buffer.write(np.ascontiguousarray(state[at]), int(slot) * per_slot)
    return buffer


@pytest.mark.parametrize("counts", [[1, 2], [50, 1]])
def test_states_far_into_the_pool(gpu, counts):
    case = Linear(counts, 2, 16, 256, 256, pool=2, slots=[0, 1])
    want, bound, states, state_bound = case.want(CHUNKS)
    per_slot = case.state[0].nbytes
    pool = (1 << 32) // per_slot + 3
    far = np.array([pool - 1, pool - 2], np.uint32)
    state = far_state(gpu, per_slot, case.state, far, pool)
    up = gpu.upload_bytes
    kw, vw, h = 2 * 256, 16 * 256, 16
    out = gpu.alloc_f32(case.tokens * vw)
    params = case.params([kw, kw, vw, h, h, vw, vw])
    params[-2] = pool
    dispatch(gpu, "attn_linear", [up(case.q), up(case.k), up(case.v), up(case.a), up(case.b), up(case.a_log), up(case.dt_bias),
                                  up(case.z), up(case.norm), up(case.starts), up(far), state, out], params)
    assert (np.abs(out.read(np.float32, want.size).reshape(want.shape) - want) <= bound).all()
    for s, slot in enumerate(far):
        got = state.read(np.float32, case.state[0].size, int(slot) * per_slot).reshape(states[0].shape)
        assert (np.abs(got - states[s]) <= state_bound[s]).all()
    # What a 32-bit offset would have met instead.
    for slot in far:
        wrapped = int(slot) * per_slot % (1 << 32)
        assert not state.read(np.float32, 1024, wrapped).any()


def test_inputs_far_into_the_pool(gpu):
    case = Conv([3, 40], 4096, 4, pool=2, slots=[0, 1])
    want, bound, states = case.want()
    per_slot = case.state[0].nbytes
    pool = (1 << 32) // per_slot + 3
    far = np.array([pool - 1, pool - 2], np.uint32)
    state = far_state(gpu, per_slot, case.state, far, pool)
    up = gpu.upload_bytes
    y = gpu.upload_f32(np.full(case.x.size, PAD, np.float32))
    dispatch(gpu, "conv_causal", [up(case.x), up(case.w), up(case.b), up(case.starts), up(far), state, y],
             [2, 43, 4096, 4, 4096, 4096, 1, 0, pool, 1])
    assert (np.abs(y.read(np.float32, case.x.size).reshape(case.x.shape) - want) <= bound).all()
    for s, slot in enumerate(far):
        assert np.array_equal(state.read(np.float32, states[0].size, int(slot) * per_slot).reshape(states[0].shape), states[s])


def test_rows_of_logits_far_apart(gpu):
    """Three rows, 2^29 floats from one to the next, of 20001 logits."""
    rng, vocab, stride = np.random.default_rng(4), 20001, (1 << 29) + 5
    logits = (2 * rng.standard_normal((3, vocab))).astype(np.float32)
    buffer = gpu.alloc(4 * (2 * stride + vocab))
    for r in range(3):
        buffer.write(logits[r], 4 * r * stride)
    up = gpu.upload_bytes
    u = rng.random(3, np.float32)
    tokens, probs = gpu.alloc(12), gpu.alloc(12)
    dispatch(gpu, "sample_logits", [buffer, up(np.full(3, 0.9, np.float32)), up(np.full(3, 30, np.uint32)),
                                    up(np.full(3, 0.8, np.float32)), up(np.zeros(3, np.float32)), up(u), tokens, probs],
             [3, vocab, stride])
    got = tokens.read(np.uint32, 3)
    for r in range(3):
        kept, share = distribution(logits[r], 0.9, 30, 0.8, 0.0)
        assert got[r] == kept[np.searchsorted(np.cumsum(share), u[r], side="right")]
