"""Sequences over a paged key-value cache, and the attention operators over them.

`Pages` keeps, on the host, which pages each sequence holds; one of it serves
all layers of a model. A step appends some tokens to some sequences (a prompt's
chunk, one token of many, a few to verify): `Pages.step` takes the pages and
gives the arrays that say where the tokens are. `Attention` holds a layer's
shape and encodes its two dispatches over a step:

    step = pages.step([(a, 200), (b, 1)]).upload(gpu)
    layer.append(cmd, step, pages, qkv, cache, positions, freqs, q_norm, k_norm)
    layer.attend(cmd, step, pages, qkv, cache, out)

include/qmr.h says what the operators compute and how a cache is laid out.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import Buffer, Command, Gpu, dispatch_layout

NO_PAGE = 0xFFFFFFFF


def f32_bits(v: float) -> int:
    return struct.unpack("<I", struct.pack("<f", v))[0]


def encode(cmd: Command, name: str, buffers: Sequence[Buffer], params: Sequence[int],
           offsets: Optional[Sequence[int]] = None) -> None:
    """Command.encode with the layout's own thread count."""
    cmd.encode(name, buffers, params, dispatch_layout(name, params)[1], 64, offsets)


@dataclass
class Step:
    """New tokens of some sequences: row s of the table, tokens
    starts[s]..starts[s+1]-1, the last of lengths[s] positions."""
    starts: np.ndarray
    lengths: np.ndarray
    table: np.ndarray
    positions: np.ndarray
    buffers: tuple[Buffer, ...] = ()

    @property
    def tokens(self) -> int:
        return int(self.starts[-1])

    @property
    def max_keys(self) -> int:
        return int(self.lengths.max())

    def upload(self, gpu: Gpu) -> "Step":
        self.buffers = tuple(gpu.upload_bytes(a) for a in (self.starts, self.lengths, self.table))
        return self


class Pages:
    """`pages` pages of `page` positions, and the sequences that hold them; a
    sequence holds at most `columns` pages."""

    def __init__(self, page: int, pages: int, columns: int):
        self.page, self.pages, self.columns = page, pages, columns
        self._free = list(range(pages - 1, -1, -1))
        self._held: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    @property
    def free(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._length[seq]

    def open(self) -> int:
        seq = self._next
        self._next += 1
        self._held[seq], self._length[seq] = [], 0
        return seq

    def close(self, seq: int) -> None:
        self._free += reversed(self._held.pop(seq))
        del self._length[seq]

    def trim(self, seq: int, length: int) -> None:
        """Forgets the positions from `length` on (tokens not accepted)."""
        if not 0 <= length <= self._length[seq]:
            raise ValueError(f"sequence {seq} holds {self._length[seq]} positions")
        keep = -(-length // self.page)
        self._free += reversed(self._held[seq][keep:])
        del self._held[seq][keep:]
        self._length[seq] = length

    def step(self, new: Sequence[tuple[int, int]]) -> Step:
        """Room for `count` more tokens of each sequence (sequence, count);
        nothing changes when the pages do not last."""
        if len({seq for seq, _ in new}) != len(new) or any(count < 0 for _, count in new):
            raise ValueError("a step names each sequence once, with its number of tokens")
        lengths = [self._length[seq] + count for seq, count in new]
        need = [-(-length // self.page) for length in lengths]
        if max(need, default=0) > self.columns:
            raise ValueError(f"a sequence holds at most {self.columns * self.page} positions")
        if sum(n - len(self._held[seq]) for n, (seq, _) in zip(need, new)) > self.free:
            raise MemoryError(f"{self.free} pages are left")
        table = np.full((len(new), self.columns), NO_PAGE, np.uint32)
        for s, (seq, _) in enumerate(new):
            held = self._held[seq]
            while len(held) < need[s]:
                held.append(self._free.pop())
            table[s, :need[s]] = held
            self._length[seq] = lengths[s]
        counts = [count for _, count in new]
        positions = [np.arange(length - count, length) for length, count in zip(lengths, counts)]
        return Step(np.cumsum([0, *counts], dtype=np.uint32), np.array(lengths, np.uint32), table,
                    np.concatenate([np.zeros(0, np.int64), *positions]).astype(np.int32))


@dataclass
class Attention:
    """One layer's shape. `rotary` dimensions of a head turn, by `sections`
    pairs an axis; eps > 0 normalises the heads of queries and keys first."""
    heads: int
    kv_heads: int
    dim: int
    rotary: int
    sections: tuple[int, ...]
    kind: str = "bf16"
    adjacent: bool = False
    dealt: bool = False
    eps: float = 0.0
    causal: bool = True
    window: int = 0
    scale: Optional[float] = None

    @property
    def width(self) -> int:
        """Floats of a token's query, key and value heads side by side."""
        return (self.heads + 2 * self.kv_heads) * self.dim

    def cache(self, gpu: Gpu, pages: Pages) -> tuple[Buffer, Buffer]:
        """Keys and values of this layer; what stands where no token was
        written reaches no row."""
        size = 2 * pages.pages * self.kv_heads * pages.page * self.dim
        return gpu.alloc(size), gpu.alloc(size)

    def append_params(self, step: Step, pages: Pages) -> list[int]:
        sections = [*self.sections, 0, 0, 0, 0][:4]
        w = self.width
        return [len(step.lengths), step.tokens, self.heads, self.kv_heads, self.dim, self.rotary, w, w, w, w,
                int(self.adjacent), int(self.dealt), len(self.sections), *sections, f32_bits(self.eps), pages.page,
                pages.pages, pages.columns]

    def append(self, cmd: Command, step: Step, pages: Pages, qkv: Buffer, cache: tuple[Buffer, Buffer],
               positions: Buffer, freqs: Buffer, q_norm: Buffer, k_norm: Buffer) -> None:
        """Turns the queries in `qkv` ([tokens][width]) in place and keeps its
        keys and values. positions: int32 [axes][tokens]."""
        k, v = 4 * self.heads * self.dim, 4 * (self.heads + self.kv_heads) * self.dim
        encode(cmd, "kv_append_rope_" + self.kind,
               [qkv, qkv, qkv, q_norm, k_norm, positions, freqs, *step.buffers, *cache, qkv],
               self.append_params(step, pages), [0, k, v, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0])

    def attend_params(self, step: Step, pages: Pages) -> list[int]:
        scale = self.dim ** -0.5 if self.scale is None else self.scale
        return [len(step.lengths), step.tokens, self.heads, self.kv_heads, self.dim, self.width, self.heads * self.dim,
                pages.page, pages.pages, pages.columns, max(step.max_keys, 1), int(self.causal), self.window,
                f32_bits(scale)]

    def attend(self, cmd: Command, step: Step, pages: Pages, qkv: Buffer, cache: tuple[Buffer, Buffer],
               out: Buffer) -> None:
        """out [tokens][heads * dim] from the queries in `qkv` and the cache."""
        encode(cmd, "attn_paged_" + self.kind, [qkv, *step.buffers, *cache, out], self.attend_params(step, pages))
