"""Inputs, 64-bit references and packed-cache helpers of the attention tests."""
from __future__ import annotations

import struct
from dataclasses import dataclass, field

import numpy as np

import qmr

HALF_MAN = {"bf16": 8, "f16": 11}  # significant bits


def f32_word(v: float) -> int:
    return struct.unpack("<I", struct.pack("<f", v))[0]


def to_half(x, kind: str) -> np.ndarray:
    """FP32 to the 16-bit patterns, nearest with ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_half(b: np.ndarray, kind: str) -> np.ndarray:
    if kind == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def pack_k(k: np.ndarray) -> np.ndarray:
    """[page][head][slot][dim] to the key blocks' order, slot by slot."""
    p, h, n, d = k.shape
    out = np.empty((p, h, n // 32, d // 8, 32, 8), k.dtype)
    for slot in range(n):
        s = slot % 32
        order = 16 * (s // 4 % 2) + 4 * (s // 8) + s % 4
        out[:, :, slot // 32, :, order, :] = k[:, :, slot].reshape(p, h, d // 8, 8)
    return out


def unpack_k(raw: np.ndarray, shape) -> np.ndarray:
    p, h, n, d = shape
    blocks = raw.reshape(p, h, n // 32, d // 8, 32, 8)
    out = np.empty(shape, raw.dtype)
    for slot in range(n):
        s = slot % 32
        order = 16 * (s // 4 % 2) + 4 * (s // 8) + s % 4
        out[:, :, slot] = blocks[:, :, slot // 32, :, order, :].reshape(p, h, d)
    return out


def pack_v(v: np.ndarray) -> np.ndarray:
    p, h, n, d = v.shape
    return np.ascontiguousarray(v.reshape(p, h, n // 8, 8, d).swapaxes(3, 4))


def unpack_v(raw: np.ndarray, shape) -> np.ndarray:
    p, h, n, d = shape
    return raw.reshape(p, h, n // 8, d, 8).swapaxes(3, 4).reshape(shape)


# ---- rotary positions ----

def axis_of(rotary: int, axes: int, dealt: bool, sections) -> np.ndarray:
    if not dealt:
        return np.repeat(np.arange(axes), sections[:axes])
    i = np.arange(rotary // 2)
    a = i % axes
    return np.where((a > 0) & (i < axes * np.asarray(sections)[a]), a, 0)


def turn64(x, positions, freqs, rotary, adjacent, axis):
    """x [tokens][heads][dim] in 64 bits with its pairs turned."""
    y = np.array(x, np.float64)
    if rotary == 0:
        return y
    t = positions.astype(np.float64)[axis].T * freqs.astype(np.float64)  # [tokens][pairs]
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    a = y[..., 0:rotary:2].copy() if adjacent else y[..., :rotary // 2].copy()
    b = y[..., 1:rotary:2].copy() if adjacent else y[..., rotary // 2:rotary].copy()
    ra, rb = a * c - b * s, b * c + a * s
    if adjacent:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = ra, rb
    else:
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = ra, rb
    return y


def pair_size(x, rotary, adjacent):
    """|a| + |b| of each element's pair (|x| where nothing turns): what an
    error of a rotation is measured against."""
    m = np.abs(np.array(x, np.float64))
    if rotary == 0:
        return m
    a = m[..., 0:rotary:2] if adjacent else m[..., :rotary // 2]
    b = m[..., 1:rotary:2] if adjacent else m[..., rotary // 2:rotary]
    s = a + b
    if adjacent:
        m[..., 0:rotary:2], m[..., 1:rotary:2] = s, s
    else:
        m[..., :rotary // 2], m[..., rotary // 2:rotary] = s, s
    return m


def rms64(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.asarray(w, np.float64)


# ---- sequences over a pool ----

@dataclass
class Batch:
    """New tokens and cache lengths of some sequences, and their pages."""
    new: list
    lengths: list
    page: int
    columns: int = 0
    spare: int = 2        # pages of the pool that no sequence names
    dropped: tuple = ()   # (sequence, column) whose page is past the pool
    seed: int = 1
    starts: np.ndarray = field(init=False)
    table: np.ndarray = field(init=False)
    pages: int = field(init=False)

    def __post_init__(self):
        need = [-(-n // self.page) for n in self.lengths]
        self.columns = max([self.columns, 1, *need])
        self.pages = sum(need) + self.spare
        order = np.random.default_rng(self.seed).permutation(self.pages)
        # Columns past a sequence's length name pages that do not exist.
        self.table = np.full((len(need), self.columns), 0xFFFFFFFF, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        for s, col in self.dropped:
            self.table[s, col] = self.pages + 7
        self.starts = np.array([0, *np.cumsum(self.new)], np.uint32)

    @property
    def tokens(self) -> int:
        return int(self.starts[-1])

    def upload(self, gpu):
        return [gpu.upload_bytes(self.starts), gpu.upload_bytes(np.array(self.lengths, np.uint32)),
                gpu.upload_bytes(self.table)]


def attend64(q, k, v, batch: Batch, scale, causal=True, window=0, max_keys=None):
    """(o, bound) [tokens][heads][dim]: the attention in 64 bits, and what its
    error is measured against (see attend_bound). k, v: [page][head][slot][dim]."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros((tokens, heads, dim)), np.zeros((tokens, heads, dim))
    for s, n in enumerate(batch.new):
        length = batch.lengths[s]
        seen_len = min(length, max_keys if max_keys is not None else length)
        col = np.arange(seen_len) // batch.page
        page = batch.table[s][col] if seen_len else np.zeros(0, np.uint32)
        held = page < batch.pages
        slot = np.arange(seen_len) % batch.page
        for i in range(n):
            pos = length - n + i
            key = np.arange(seen_len)
            seen = held & ((key <= pos) if causal else (key >= 0))
            if window:
                seen = seen & (key > pos - window)
            if not seen.any():
                continue
            at = np.flatnonzero(seen)
            for h in range(heads):
                kk = k[page[at], h // group, slot[at]]
                vv = v[page[at], h // group, slot[at]]
                qq = q[int(batch.starts[s]) + i, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    x = kk @ qq * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[batch.starts[s] + i, h] = p @ vv
                    size = (np.abs(kk) @ np.abs(qq) * scale).max()
                    bound[batch.starts[s] + i, h] = attend_bound(size, len(at)) * (p @ np.abs(vv))
    return out, bound


def attend_bound(size: float, keys: int) -> float:
    """Relative to sum p|v|. A score is off by at most 2e-6 of `size` =
    scale * sum |q k| (two f16 terms keep 22 bits, 2.4e-7; up to 24 + 5 adds
    of 6e-8 each), which moves p by that much and the sum of all p by no
    more: twice. Sums over blocks of 32 keys: their roundings, 1.2e-7 each,
    add up as a random walk's. 1e-6 for the exponential, the weights' terms
    and the division."""
    return 2 * 2e-6 * size + 2.4e-7 * np.sqrt(keys / 32) + 1e-6


def make_pool(batch: Batch, kv_heads: int, dim: int, kind: str, rng, fill=0x7F80):
    """Key and value bit patterns [page][head][slot][dim]; slots that no
    sequence holds are filled with `fill` (an infinity of bf16, a NaN of f16)."""
    shape = (batch.pages, kv_heads, batch.page, dim)
    k, v = (to_half(rng.standard_normal(shape), kind) for _ in range(2))
    used = np.zeros((batch.pages, batch.page), bool)
    for s, length in enumerate(batch.lengths):
        for col in range(-(-length // batch.page)):
            if batch.table[s, col] < batch.pages:
                used[batch.table[s, col], :max(0, min(batch.page, length - col * batch.page))] = True
    hole = ~used[:, None, :, None] & np.ones(shape, bool)
    k[hole], v[hole] = fill, fill
    return k, v


def attend(gpu: "qmr.Gpu", kind, q, kb, vb, batch: Batch, scale, causal=True, window=0, max_keys=None, pad=0, shift=0,
           static=False):
    """One attn_paged dispatch over the bit patterns kb, vb; rows `pad` floats
    longer than their heads, views `shift` floats into their buffers."""
    tokens, heads, dim = q.shape
    width = heads * dim
    rows = np.full((tokens, width + pad), np.nan, np.float32)
    rows[:, :width] = q.reshape(tokens, width)
    qb = gpu.upload_f32(np.concatenate([np.zeros(shift, np.float32), rows.ravel()]))
    y = gpu.upload_f32(np.full(shift + tokens * (width + pad), 77.0, np.float32))
    params = [len(batch.new), tokens, heads, kb.shape[1], dim, width + pad, width + pad, batch.page, batch.pages,
              batch.columns, max_keys or batch.columns * batch.page, int(causal), window, f32_word(scale)]
    name = "attn_paged_" + kind
    _, threads = qmr.dispatch_layout(name, params)
    cmd = gpu.begin()
    cmd.encode(name, [qb, *batch.upload(gpu), gpu.upload_bytes(pack_k(kb)), gpu.upload_bytes(pack_v(vb)), y], params,
               threads, 64, [4 * shift, 0, 0, 0, 0, 0, 4 * shift], static_scratch=static)
    cmd.finish()
    got = y.read(np.float32, shift + tokens * (width + pad))
    assert (got[:shift] == 77.0).all()
    got = got[shift:].reshape(tokens, width + pad)
    assert (got[:, width:] == 77.0).all(), "written past the rows"
    return got[:, :width].reshape(tokens, heads, dim)


def check_attend(got, want, bound, what=""):
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    off = np.abs(got - want) - bound
    off = np.where(np.isnan(off), 0.0, off)
    i = np.unravel_index(int(np.argmax(off)), off.shape)
    assert off[i] <= 0, f"{what}: {i}: {got[i]} vs {want[i]}, bound {bound[i]:.3e}; {(off > 0).sum()} of {off.size} off"
