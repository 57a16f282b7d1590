"""Linear attention and the causal convolution in 64 bits, with bounds on the
error of 32, and dispatches of both over rows with padding around them."""
from __future__ import annotations

import struct

import numpy as np

ULP = 2.0 ** -24  # half a step of FP32, relative
FRESH = 1 << 31
PAD = 9.0  # what stands around rows, before and after


def f32_word(v: float) -> int:
    return struct.unpack("<I", struct.pack("<f", v))[0]


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def owners(slots, pool):
    """Of each sequence its slot, or None: past the pool, or named before."""
    seen, out = set(), []
    for word in slots:
        slot = int(word) % FRESH
        out.append(slot if slot < pool and slot not in seen else None)
        if slot < pool:
            seen.add(slot)
    return out


class Rows:
    """FP32 rows of `width` in a buffer, `shift` floats before the first and
    `pad` behind each."""

    def __init__(self, gpu, x, pad=0, shift=0):
        x = np.asarray(x, np.float32)
        self.tokens, self.width, self.pad, self.shift = x.shape[0], x.shape[1], pad, shift
        rows = np.full((self.tokens, self.width + pad), PAD, np.float32)
        rows[:, :self.width] = x
        self.buffer = gpu.upload_f32(np.concatenate([np.full(shift, PAD, np.float32), rows.ravel()]))

    @property
    def stride(self):
        return self.width + self.pad

    @property
    def offset(self):
        return 4 * self.shift

    def read(self):
        """The rows; what stands around them has to be untouched."""
        got = self.buffer.read(np.float32, self.shift + self.tokens * self.stride)
        assert (got[:self.shift] == PAD).all()
        got = got[self.shift:].reshape(self.tokens, self.stride)
        assert (got[:, self.width:] == PAD).all()
        return got[:, :self.width]


class Linear:
    """One attn_linear dispatch and what it has to leave."""

    def __init__(self, counts, k_heads=2, v_heads=4, dk=32, dv=32, *, gates=True, delta=True, qk_eps=1e-6, out_eps=1e-6,
                 fixed=False, keep=True, slots=None, pool=None, behind=0, most=None, seed=0):
        rng = np.random.default_rng(seed + 1000 * sum(counts) + dk)
        self.counts, self.tokens = list(counts), sum(counts) + behind
        self.k_heads, self.v_heads, self.dk, self.dv = k_heads, v_heads, dk, dv
        self.gates, self.delta, self.qk_eps, self.out_eps, self.keep = gates, delta, qk_eps, out_eps, keep
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
        self.pool = pool or len(counts) + 2
        self.slots = np.asarray(rng.permutation(self.pool)[:len(counts)] if slots is None else slots, np.uint32)
        self.most = most or max(*counts, 1)
        n, f = self.tokens, np.float32
        size = 1.0 if qk_eps else 1 / np.sqrt(dk) / 1.5  # keys at most about 1 long
        self.q, self.k = ((rng.standard_normal((n, k_heads * dk)) * size).astype(f) for _ in range(2))
        if not qk_eps:
            k = self.k.reshape(n, k_heads, dk)
            k /= np.maximum(1, np.linalg.norm(k, axis=-1, keepdims=True) * f(1 + 1e-6))
        self.v = rng.standard_normal((n, v_heads * dv)).astype(f)
        self.a = rng.standard_normal((1 if fixed else n, v_heads)).astype(f)
        if not gates:
            self.a = np.log(rng.uniform(0.6, 0.999, self.a.shape)).astype(f)
        self.fixed = fixed
        self.b = (2 * rng.standard_normal((n, v_heads))).astype(f)
        self.a_log = np.log(rng.uniform(1, 16, v_heads)).astype(f)
        self.dt_bias = np.log(np.expm1(np.exp(rng.uniform(np.log(1e-3), np.log(0.1), v_heads)))).astype(f)
        self.z = rng.standard_normal((n, v_heads * dv)).astype(f)
        self.norm = rng.uniform(0.5, 1.5, dv).astype(f)
        self.state = rng.standard_normal((self.pool, v_heads, dk, dv)).astype(f)
        self.scale = np.float32(1 / np.sqrt(dk))

    def params(self, strides):
        return [len(self.counts), self.tokens, self.k_heads, self.v_heads, self.dk, self.dv, *strides, self.most,
                int(self.gates), int(self.delta), f32_word(float(self.scale)), f32_word(self.qk_eps), f32_word(self.out_eps),
                self.pool, int(self.keep)]

    def run(self, gpu, pad=0, shift=0, static=False):
        """(out rows, states) of a dispatch on the arrays as they are now."""
        rows = [Rows(gpu, x, pad, shift) for x in (self.q, self.k, self.v, self.a, self.b, self.z)]
        q, k, v, a, b, z = rows
        out = Rows(gpu, np.full((self.tokens, self.v_heads * self.dv), PAD), pad, shift)
        state = gpu.upload_f32(np.concatenate([np.full(shift, PAD, np.float32), self.state.ravel()]))
        up = gpu.upload_bytes
        buffers = [q.buffer, k.buffer, v.buffer, a.buffer, b.buffer, up(self.a_log), up(self.dt_bias), z.buffer,
                   up(self.norm), up(self.starts), up(self.slots), state, out.buffer]
        offsets = [q.offset, k.offset, v.offset, a.offset, b.offset, 0, 0, z.offset, 0, 0, 0, 4 * shift, out.offset]
        strides = [q.stride, k.stride, v.stride, 0 if self.fixed else a.stride, b.stride, z.stride, out.stride]
        dispatch(gpu, "attn_linear", buffers, self.params(strides), offsets, static)
        after = state.read(np.float32, shift + self.state.size)
        assert (after[:shift] == PAD).all()
        return out.read(), after[shift:].reshape(self.state.shape)

    def want(self, roundings, floor=0.0):
        """(out, its bound, states, their bound) in 64 bits. Of a column of the
        state the error's length grows by `roundings` of what a token leaves
        there, and shrinks by its decay: the step is a contraction, since keys
        are at most 1 long and beta below 1. A token's part may also be off by
        `floor` of the largest value of its column among the 32 tokens (from the
        sequence's first on) that it is one of."""
        hk, hv, dk, dv = self.k_heads, self.v_heads, self.dk, self.dv
        d = np.float64
        out = np.full((self.tokens, hv * dv), PAD)
        bound = np.zeros((self.tokens, hv, dv))
        states, state_bound = self.state.astype(d), np.zeros(self.state.shape)
        head = np.arange(hv) // (hv // hk)
        for s, slot in enumerate(owners(self.slots, self.pool)):
            first, n = int(self.starts[s]), min(self.counts[s], self.most)
            fresh = self.slots[s] >= FRESH or slot is None
            S = np.zeros((hv, dk, dv)) if fresh else self.state[slot].astype(d)
            E = np.zeros((hv, dv))
            for t in range(first, first + n):
                q, k = self.q[t].reshape(hk, dk).astype(d), self.k[t].reshape(hk, dk).astype(d)
                if self.qk_eps:
                    q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + self.qk_eps) for x in (q, k))
                q, k, v = q[head] * d(self.scale), k[head], self.v[t].reshape(hv, dv).astype(d)
                g = self.a[0 if self.fixed else t].astype(d)
                # The decay's own error: a rounded exponent, worth |g| of it.
                if self.gates:
                    g = -np.exp(self.a_log.astype(d)) * np.logaddexp(0, g + self.dt_bias.astype(d))
                decay = np.exp(g)[:, None, None]
                slip = (4 * np.abs(np.where(np.isfinite(g), g, 0)) + 4)[:, None] * ULP
                S = decay * S
                size = np.linalg.norm(S, axis=1)
                beta = sigmoid(self.b[t].astype(d))[:, None] if self.delta else 1.0
                u = beta * (v - np.einsum("hij,hi->hj", S, k)) if self.delta else v
                S = S + k[:, :, None] * u[:, None, :]
                length = np.linalg.norm(k, axis=-1)[:, None]
                at = first + (t - first) // 32 * 32
                largest = np.abs(self.v[at:min(at + 32, first + n)]).max(0).reshape(hv, dv).astype(d)
                E = decay[:, 0] * E + floor * length * largest + roundings * ULP * (size + length * (np.abs(u) + np.abs(v))) + 2 * slip * size
                o = np.einsum("hij,hi->hj", S, q)
                off = np.linalg.norm(q, axis=-1)[:, None] * (E + roundings * ULP * np.linalg.norm(S, axis=1))
                if self.out_eps:
                    z = self.z[t].reshape(hv, dv).astype(d)
                    rms = np.sqrt((o * o).mean(-1, keepdims=True) + self.out_eps)
                    by = self.norm.astype(d) * z * sigmoid(z) / rms
                    off = np.abs(by) * (off + np.abs(o) * (np.linalg.norm(off, axis=-1, keepdims=True) / np.sqrt(dv) / rms
                                                           + 40 * ULP))
                    o = o * by
                out[t] = o.ravel()
                bound[t] = off
            if slot is not None and self.keep and n > 0:
                states[slot] = S
                state_bound[slot] = E[:, None, :]
        return out, bound.reshape(self.tokens, hv * dv), states, state_bound

    def check(self, gpu, roundings, where="", **how):
        got, after = self.run(gpu, **how)
        want, bound, states, state_bound = self.want(roundings)
        off = np.abs(got - want)
        assert np.isfinite(got).all(), where
        assert (off <= bound).all(), (where, float((off / np.maximum(bound, 1e-300)).max()))
        off = np.abs(after - states)
        assert (off <= state_bound).all(), (where, "state", float((off / np.maximum(state_bound, 1e-300)).max()))
        return got, after


class Conv:
    """One conv_causal dispatch and what it has to leave."""

    def __init__(self, counts, channels=8, width=4, *, silu=True, bias=False, keep=True, slots=None, pool=None, behind=0,
                 seed=0):
        rng = np.random.default_rng(seed + 1000 * sum(counts) + channels)
        self.counts, self.tokens, self.channels, self.width = list(counts), sum(counts) + behind, channels, width
        self.silu, self.bias, self.keep = silu, bias, keep
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
        self.pool = pool or len(counts) + 2
        self.slots = np.asarray(rng.permutation(self.pool)[:len(counts)] if slots is None else slots, np.uint32)
        self.x = rng.standard_normal((self.tokens, channels)).astype(np.float32)
        self.w = rng.standard_normal((channels, width)).astype(np.float32)
        self.b = rng.standard_normal(channels).astype(np.float32)
        self.state = rng.standard_normal((self.pool, width - 1, channels)).astype(np.float32)

    def run(self, gpu, pad=0, shift=0, static=False):
        x, y = Rows(gpu, self.x, pad, shift), Rows(gpu, np.full(self.x.shape, PAD), pad, shift)
        state = gpu.upload_f32(np.concatenate([np.full(shift, PAD, np.float32), self.state.ravel()]))
        up = gpu.upload_bytes
        dispatch(gpu, "conv_causal", [x.buffer, up(self.w), up(self.b), up(self.starts), up(self.slots), state, y.buffer],
                 [len(self.counts), self.tokens, self.channels, self.width, x.stride, y.stride, int(self.silu),
                  int(self.bias), self.pool, int(self.keep)], [x.offset, 0, 0, 0, 0, 4 * shift, y.offset], static)
        after = state.read(np.float32, shift + self.state.size)
        assert (after[:shift] == PAD).all()
        return y.read(), after[shift:].reshape(self.state.shape)

    def want(self):
        """(y, its bound, states) in 64 bits. A sum of width products and the
        bias rounds once each; SiLU has a slope of at most 1.1, and rounds in
        its exponential (2), sum, quotient."""
        w, n = self.width, self.channels
        y, bound, states = np.full((self.tokens, n), PAD), np.zeros((self.tokens, n)), self.state.copy()
        for s, slot in enumerate(owners(self.slots, self.pool)):
            first, count = int(self.starts[s]), self.counts[s]
            fresh = self.slots[s] >= FRESH or slot is None
            old = np.zeros((w - 1, n), np.float32) if fresh else self.state[slot]
            rows = np.concatenate([old, self.x[first:first + count]])
            for t in range(count):
                part = rows[t:t + w].T.astype(np.float64) * self.w
                sum_ = part.sum(1) + (self.b if self.bias else 0)
                off = (w + 1) * ULP * (np.abs(part).sum(1) + (np.abs(self.b) if self.bias else 0))
                if self.silu:
                    sum_ = sum_ * sigmoid(sum_)
                    off = 1.1 * off + 6 * ULP * np.abs(sum_)
                y[first + t], bound[first + t] = sum_, off
            if slot is not None and self.keep and count:
                states[slot] = rows[count:]
        return y, bound, states

    def check(self, gpu, **how):
        got, after = self.run(gpu, **how)
        want, bound, states = self.want()
        assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())
        assert np.array_equal(after, states)
        return got, after


def dispatch(gpu, name, buffers, params, offsets=None, static=False):
    import qmr

    cmd = gpu.begin()
    try:
        cmd.encode(name, buffers, params, qmr.dispatch_layout(name, params)[1], 64, offsets, static_scratch=static)
        cmd.finish()
    finally:
        cmd.release()
