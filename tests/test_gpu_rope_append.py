"""rope_axes and kv_append_rope against their definitions in 64 bits."""
import numpy as np
import pytest

import qmr
from attention_cases import (HALF_MAN, Batch, axis_of, f32_word, from_half, pack_k, pack_v, pair_size, rms64, to_half,
                             turn64, unpack_k, unpack_v)

pytestmark = pytest.mark.gpu

EPS = 1e-6
# A turn's error against |a| + |b|: 1.9e-7 from the fraction of a turn (2^-25
# of one), 2.4e-7 from sine and cosine (two ulp), 1.2e-7 from the products and
# their sum.
TURN = 6e-7
# The norm before it: 14 adds in the sum of squares, the mean, the root, the
# quotient and two products, 6e-8 each.
NORM = 1.3e-6


def freqs_of(rotary, base=1e4):
    return (base ** (-np.arange(0, rotary, 2) / max(rotary, 1))).astype(np.float32)


def positions_of(rng, axes, tokens):
    p = rng.integers(0, 70000, (max(axes, 1), tokens)).astype(np.int32)
    p[0, 0] = 1_048_575
    p[-1, -1] = -3
    return p


ROPES = [  # dim, rotary, adjacent, dealt, sections
    (64, 64, 0, 0, [32, 0, 0, 0]), (256, 64, 0, 1, [11, 11, 10, 0]), (256, 256, 1, 0, [128, 0, 0, 0]),
    (72, 72, 0, 0, [18, 18, 0, 0]), (128, 100, 0, 0, [20, 10, 20, 0]), (6, 4, 1, 0, [1, 1, 0, 0]),
    (250, 250, 0, 0, [60, 0, 5, 60]), (128, 64, 1, 1, [8, 8, 8, 8]), (2, 2, 0, 0, [1, 0, 0, 0]),
    (80, 24, 0, 1, [12, 0, 0, 0]),
]


@pytest.mark.parametrize("dim,rotary,adjacent,dealt,sections", ROPES)
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 24), (7, 5), (300, 3)])
def test_rope_axes(gpu, dim, rotary, adjacent, dealt, sections, tokens, heads):
    rng = np.random.default_rng(dim + tokens)
    axes = max(i for i in range(4) if sections[i]) + 1
    x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    pos, freqs = positions_of(rng, axes, tokens), freqs_of(rotary)
    want = turn64(x, pos, freqs, rotary, adjacent, axis_of(rotary, axes, dealt, sections))
    for pad, shift, in_place in ((0, 0, False), (4, 4, True), (3, 1, False), (1, 3, True)):
        width = heads * dim
        rows = np.full((tokens, width + pad), 9.0, np.float32)
        rows[:, :width] = x.reshape(tokens, width)
        xb = gpu.upload_f32(np.concatenate([np.full(shift, 9.0, np.float32), rows.ravel()]))
        yb = xb if in_place else gpu.upload_f32(np.full(shift + rows.size, 9.0, np.float32))
        gpu.dispatch("rope_axes", [xb, gpu.upload_bytes(pos), gpu.upload_f32(freqs), yb],
                     [tokens, heads, dim, rotary, width + pad, width + pad, adjacent, dealt, axes, *sections],
                     offsets=[4 * shift, 0, 0, 4 * shift], group_size=64)
        got = yb.read(np.float32, shift + rows.size)
        assert (got[:shift] == 9).all()
        got = got[shift:].reshape(tokens, width + pad)
        assert (got[:, width:] == 9).all()
        got = got[:, :width].reshape(tokens, heads, dim)
        assert (np.abs(got - want) <= TURN * pair_size(x, rotary, adjacent)).all()
        assert np.array_equal(got[..., rotary:], x[..., rotary:])


def test_a_turn_keeps_lengths_and_differences(gpu):
    # q and k turned by positions p and p + d have the same product for any p.
    rng = np.random.default_rng(2)
    x = np.repeat(rng.standard_normal((1, 2, 64)), 40, axis=0).astype(np.float32)
    pos = np.stack([np.arange(40) * 2500, np.arange(40) * 2500], axis=0).astype(np.int32)
    out = []
    for d in (0, 17):
        y = gpu.alloc_f32(x.size)
        gpu.dispatch("rope_axes", [gpu.upload_f32(x.ravel()), gpu.upload_bytes((pos + d).astype(np.int32)),
                                   gpu.upload_f32(freqs_of(64)), y],
                     [40, 2, 64, 64, 128, 128, 0, 0, 2, 16, 16, 0, 0], group_size=64)
        out.append(gpu.read_f32(y, x.size).reshape(x.shape).astype(np.float64))
    dots = (out[0][:, 0] * out[1][:, 1]).sum(-1)
    size = np.abs(x[0, 0]).sum() * np.abs(x[0, 1]).max()
    assert np.abs(dots - dots[0]).max() <= 4 * TURN * size


class Append:
    """One kv_append_rope dispatch and what it has to leave."""

    def __init__(self, kind, batch, heads, kv_heads, dim, rotary, adjacent=0, dealt=0, sections=None, norm=False,
                 seed=0, pad=0, shift=0):
        self.__dict__.update(locals())
        rng = np.random.default_rng(seed)
        self.sections = sections or [rotary // 2, 0, 0, 0]
        self.axes = 0 if rotary == 0 else max(i for i in range(4) if self.sections[i]) + 1
        t = batch.tokens
        self.q, self.k, self.v = (rng.standard_normal((t, h, dim)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
        self.pos = positions_of(rng, self.axes, t)
        self.freqs = freqs_of(rotary)
        self.wq, self.wk = ((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
        shape = (batch.pages, kv_heads, batch.page, dim)
        self.old_k, self.old_v = (to_half(rng.standard_normal(shape), kind) for _ in range(2))

    def params(self):
        w = self.width
        return [len(self.batch.new), self.batch.tokens, self.heads, self.kv_heads, self.dim, self.rotary, w, w, w, w,
                self.adjacent, self.dealt, self.axes, *self.sections, f32_word(EPS) if self.norm else 0,
                self.batch.page, self.batch.pages, self.batch.columns]

    def run(self, gpu, in_place=False):
        t, hq, hk, dim = self.batch.tokens, self.heads, self.kv_heads, self.dim
        self.width = (hq + 2 * hk) * dim + self.pad
        rows = np.full((t, self.width), 5.0, np.float32)
        rows[:, :(hq + 2 * hk) * dim] = np.concatenate([x.reshape(t, -1) for x in (self.q, self.k, self.v)], axis=1)
        qkv = gpu.upload_f32(np.concatenate([np.full(self.shift, 5.0, np.float32), rows.ravel()]))
        out = qkv if in_place else gpu.upload_f32(np.full(self.shift + rows.size, 5.0, np.float32))
        kc, vc = gpu.upload_bytes(pack_k(self.old_k)), gpu.upload_bytes(pack_v(self.old_v))
        at = 4 * self.shift
        gpu.dispatch("kv_append_rope_" + self.kind,
                     [qkv, qkv, qkv, gpu.upload_f32(self.wq), gpu.upload_f32(self.wk), gpu.upload_bytes(self.pos),
                      gpu.upload_f32(self.freqs), *self.batch.upload(gpu), kc, vc, out], self.params(),
                     offsets=[at, at + 4 * hq * dim, at + 4 * (hq + hk) * dim, 0, 0, 0, 0, 0, 0, 0, 0, 0, at],
                     group_size=64)
        shape = self.old_k.shape
        got = out.read(np.float32, self.shift + rows.size)[self.shift:].reshape(t, self.width)
        rest = rows[:, hq * dim:] if in_place else np.full((t, self.width - hq * dim), 5.0)
        assert np.array_equal(got[:, hq * dim:], rest)
        return (got[:, :hq * dim].reshape(t, hq, dim), unpack_k(kc.read(np.uint16, self.old_k.size), shape),
                unpack_v(vc.read(np.uint16, self.old_v.size), shape))

    def check(self, gpu, **how):
        q, kc, vc = self.run(gpu, **how)
        axis = axis_of(self.rotary, self.axes, self.dealt, self.sections)

        def turned(x, w):
            x = rms64(x, w, float(np.float32(EPS))) if self.norm else x.astype(np.float64)
            size = pair_size(x, self.rotary, self.adjacent)
            return turn64(x, self.pos, self.freqs, self.rotary, self.adjacent, axis), \
                size * (TURN + (NORM if self.norm else 0))

        want, bound = turned(self.q, self.wq)
        assert (np.abs(q - want) <= bound).all()
        want, bound = turned(self.k, self.wk)
        left_k, left_v = self.old_k.copy(), self.old_v.copy()
        b = self.batch
        for s, n in enumerate(b.new):
            for i in range(n):
                pos, t = b.lengths[s] - n + i, int(b.starts[s]) + i
                if pos < 0 or pos >= b.columns * b.page or b.table[s, pos // b.page] >= b.pages:
                    continue
                page, slot = b.table[s, pos // b.page], pos % b.page
                got = from_half(kc[page, :, slot], self.kind)
                half = np.abs(want[t]) * 2.0 ** -HALF_MAN[self.kind] + 2.0 ** -25
                assert (np.abs(got - want[t]) <= half + 1.01 * bound[t]).all()
                left_k[page, :, slot] = kc[page, :, slot]
                left_v[page, :, slot] = to_half(self.v[t], self.kind)
        assert np.array_equal(kc, left_k), "a slot that no new token has was written"
        assert np.array_equal(vc, left_v)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,adjacent,dealt,sections", [
    (6, 2, 64, 64, 0, 0, None), (24, 4, 256, 64, 0, 1, [11, 11, 10, 0]), (3, 1, 72, 72, 1, 0, [18, 18, 0, 0]),
    (5, 5, 128, 100, 0, 0, None), (2, 1, 8, 2, 0, 0, None), (4, 2, 80, 0, 0, 0, [0, 0, 0, 0]), (0, 3, 192, 192, 0, 0, None)])
def test_append(gpu, kind, norm, heads, kv_heads, dim, rotary, adjacent, dealt, sections):
    for new, lengths in (([1], [1]), ([1, 1, 1], [5, 32, 33]), ([0, 7, 30, 1], [9, 40, 30, 128])):
        Append(kind, Batch(new, lengths, 32, seed=dim), heads, kv_heads, dim, rotary, adjacent, dealt, sections, norm,
               seed=dim).check(gpu)


@pytest.mark.parametrize("pad,shift,in_place", [(0, 0, True), (4, 4, True), (3, 0, False), (1, 1, True), (2, 3, False)])
def test_strides_offsets_and_place(gpu, pad, shift, in_place):
    for norm in (False, True):
        Append("bf16", Batch([3, 20], [50, 41], 32), 4, 2, 64, 32, norm=norm, pad=pad, shift=shift).check(
            gpu, in_place=in_place)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_every_place_in_a_chunk(gpu, kind):
    for old in range(9):
        for new in (1, 2, 7, 8, 9, 17):
            Append(kind, Batch([new], [old + new], 32, seed=old), 1, 1, 16, 16, seed=new).check(gpu)


def test_many_sequences(gpu):
    rng = np.random.default_rng(4)
    new = [int(n) for n in rng.integers(0, 3, 200)]
    Append("f16", Batch(new, [n + int(o) for n, o in zip(new, rng.integers(0, 40, 200))], 32), 2, 1, 64, 64).check(gpu)


def test_tokens_without_a_place(gpu):
    # Positions before the first, past the table's columns, and in pages past
    # the pool are dropped; the others are kept.
    b = Batch([6, 5, 40], [3, 36, 64], 32, dropped=((2, 1),))
    b.lengths[1] = 70  # its new tokens are positions 65..69: two columns hold 64
    Append("bf16", b, 2, 1, 64, 64).check(gpu)


def test_values_out_of_range(gpu):
    a = Append("f16", Batch([9], [9], 32), 1, 1, 16, 0, sections=[0, 0, 0, 0])
    a.v[3, 0, :4] = [1e6, -1e6, np.inf, 65519.0]
    a.k[3, 0, :4] = [1e6, -1e6, np.inf, 65519.0]
    _, k, v = a.run(gpu)
    page = a.batch.table[0, 0]
    for c in (k, v):
        assert list(from_half(c[page, 0, 3, :4], "f16")) == [np.inf, -np.inf, np.inf, 65504.0]


def test_refusals(gpu):
    b = Batch([2], [40], 32)
    a = Append("f16", b, 2, 1, 64, 64)
    a.run(gpu)
    f, cache = gpu.alloc_f32(4096), gpu.alloc(2 * b.pages * 32 * 64 + 64)
    pos, freq = gpu.upload_bytes(a.pos), gpu.upload_f32(a.freqs)
    bufs = [f, f, f, f, f, pos, freq, *b.upload(gpu), cache, gpu.alloc(2 * b.pages * 32 * 64), gpu.alloc_f32(1024)]
    offs = [0, 512, 768] + [0] * 10

    def refused(match, buffers=bufs, offsets=offs, params=None):
        with pytest.raises(qmr.QmrError, match=match):
            gpu.dispatch("kv_append_rope_f16", buffers, params or a.params(), offsets=offsets, group_size=64)

    refused("16-byte aligned", offsets=[*offs[:10], 4, 0, 0])
    refused("overlaps input buffer 10", buffers=[*bufs[:11], cache, bufs[12]])
    refused("overlaps input buffer 0", buffers=[cache, *bufs[1:]])
    refused("overlaps input buffer 0", buffers=[*bufs[:12], f], offsets=[*offs[:12], 4])
    refused("overlaps input buffer 1", buffers=[*bufs[:12], f], offsets=[*offs[:12], 512])
    refused("ends at", buffers=[*bufs[:12], gpu.alloc_f32(4)])
    with pytest.raises(qmr.QmrError, match="overlaps input buffer 0"):
        gpu.dispatch("rope_axes", [f, pos, freq, f], [2, 2, 64, 64, 128, 132, 0, 0, 1, 32, 0, 0, 0], group_size=64)
