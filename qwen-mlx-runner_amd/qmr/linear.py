"""Sequences with states of linear attention, its operators, and drawing tokens.

`Slots` keeps, on the host, which slot of a layer's states each sequence has;
one of it serves all layers of a model. `Slots.step` gives the arrays that say
where a step's tokens are. `Layer` holds a layer's shape and encodes its two
dispatches over a step; `Draws` holds what a row of logits is drawn with:

    step = slots.step([(a, 200), (b, 1)]).upload(gpu)
    layer.convolve(cmd, step, slots, rows, filters, bias, states, qkv)
    layer.attend(cmd, step, slots, rows, qkv, weights, states, out)
    draws.sample(cmd, logits, vocab, tokens, probs)

Single tokens go faster in a step of their own than beside a prompt's, in the same
command. A sequence has one state, of its last token: what a token did to it is not
undone. Tokens that may be taken back (to verify) go in a step with keep=False,
and the accepted ones again in one with keep=True. A step that not every layer ran,
since a call was refused or its command failed, is given to `Slots.undo` (a
layer's own two calls do that when they are refused). include/qmr.h says what the
operators compute.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass
from typing import NamedTuple, Optional, Sequence

import numpy as np

from . import Buffer, Command, Gpu
from .paged import encode, f32_bits

FRESH = 1 << 31
NO_TOKEN = 0xFFFFFFFF


@dataclass
class Step:
    """New tokens of some sequences: tokens starts[s]..starts[s+1]-1 are those
    of the sequence whose states are in slot words[s], where what they make of
    them is kept or not. `begun` are the sequences that have their first tokens
    kept by it."""
    starts: np.ndarray
    words: np.ndarray
    keep: bool = True
    buffers: tuple[Buffer, ...] = ()
    begun: frozenset[int] = frozenset()

    @property
    def tokens(self) -> int:
        return int(self.starts[-1])

    @property
    def most(self) -> int:
        return max(int(np.diff(self.starts.astype(np.int64)).max()), 1)

    def upload(self, gpu: Gpu) -> "Step":
        self.buffers = tuple(gpu.upload_bytes(a) for a in (self.starts, self.words))
        return self


class Slots:
    """`slots` states of each layer, and the sequences that have them."""

    def __init__(self, slots: int):
        if not 0 < slots < FRESH:
            raise ValueError("a pool has 1 to 2^31 - 1 slots")
        self.slots = slots
        self._free = list(range(slots - 1, -1, -1))
        self._held: dict[int, int] = {}
        self._fresh: set[int] = set()
        self._begun: dict[int, Step] = {}  # sequences whose one kept step so far this is
        self._next = 0

    @property
    def free(self) -> int:
        return len(self._free)

    def open(self) -> int:
        if not self._free:
            raise MemoryError("no slot is left")
        seq = self._next
        self._next += 1
        self._held[seq] = self._free.pop()
        self._fresh.add(seq)
        return seq

    def close(self, seq: int) -> None:
        self._free.append(self._held.pop(seq))
        self._fresh.discard(seq)
        self._begun.pop(seq, None)

    def step(self, new: Sequence[tuple[int, int]], keep: bool = True) -> Step:
        """`count` more tokens of each sequence (sequence, count). A sequence's
        first tokens find zeros, whatever the slot's last owner left. A step that
        keeps is to be run by every layer, once."""
        if not new or len({seq for seq, _ in new}) != len(new) or any(count < 0 for _, count in new):
            raise ValueError("a step names each sequence once, with its number of tokens")
        words = [self._held[seq] | (FRESH if seq in self._fresh else 0) for seq, _ in new]
        kept = {seq for seq, count in new if keep and count > 0}
        step = Step(np.cumsum([0, *(count for _, count in new)], dtype=np.uint32), np.array(words, np.uint32), keep,
                    begun=frozenset(kept & self._fresh))
        self._fresh -= kept
        for seq in kept:
            self._begun.pop(seq, None)
        self._begun.update(dict.fromkeys(step.begun, step))
        return step

    def undo(self, step: Step) -> None:
        """Takes back a step that not every layer ran: the sequences whose first
        tokens it has start from zeros again, whatever it left in their slots. The
        states of its other sequences are as far as each layer ran, which nothing
        brings back."""
        again = {seq for seq in step.begun if self._begun.get(seq) is step}
        self._fresh |= again
        for seq in again:
            del self._begun[seq]


@contextmanager
def _undone(slots: Slots, step: Step):
    """Takes the step back if what is inside is refused."""
    try:
        yield
    except BaseException:
        slots.undo(step)
        raise


class Weights(NamedTuple):
    """A layer's small weights: a_log and dt_bias [v_heads], norm [dv]."""
    a_log: Buffer
    dt_bias: Buffer
    norm: Buffer


class States(NamedTuple):
    """Of all slots: a layer's last inputs, and its heads' states."""
    inputs: Buffer
    heads: Buffer


@dataclass
class Layer:
    """One layer's shape. Its input product's rows hold queries, keys and values
    (`channels`), the output gates z, and b and a of each value head; the
    convolution takes the channels of `width` tokens."""
    k_heads: int
    v_heads: int
    dk: int
    dv: int
    width: int = 4
    bias: bool = False
    qk_eps: float = 1e-6
    out_eps: float = 1e-6
    scale: Optional[float] = None

    @property
    def channels(self) -> int:
        return 2 * self.k_heads * self.dk + self.v_heads * self.dv

    @property
    def row(self) -> int:
        """Floats of a token's row: channels, z, b, a."""
        return self.channels + self.out_width + 2 * self.v_heads

    @property
    def out_width(self) -> int:
        return self.v_heads * self.dv

    def states(self, gpu: Gpu, slots: Slots) -> States:
        """Of this layer; nothing of them is read before it is written."""
        return States(gpu.alloc_f32(slots.slots * (self.width - 1) * self.channels),
                      gpu.alloc_f32(slots.slots * self.v_heads * self.dk * self.dv))

    def convolve_params(self, step: Step, slots: Slots) -> list[int]:
        return [len(step.words), step.tokens, self.channels, self.width, self.row, self.channels, 1, int(self.bias),
                slots.slots, int(step.keep)]

    def convolve(self, cmd: Command, step: Step, slots: Slots, rows: Buffer, filters: Buffer, bias: Buffer,
                 states: States, qkv: Buffer) -> None:
        """qkv [tokens][channels] from the product's rows [tokens][row]; `bias`
        is read if the layer has one, and may be any buffer if not."""
        with _undone(slots, step):
            encode(cmd, "conv_causal", [rows, filters, bias, *step.buffers, states.inputs, qkv],
                   self.convolve_params(step, slots))

    def attend_params(self, step: Step, slots: Slots) -> list[int]:
        scale = self.dk ** -0.5 if self.scale is None else self.scale
        c, r = self.channels, self.row
        return [len(step.words), step.tokens, self.k_heads, self.v_heads, self.dk, self.dv, c, c, c, r, r, r, self.out_width,
                step.most, 1, 1, f32_bits(scale), f32_bits(self.qk_eps), f32_bits(self.out_eps), slots.slots,
                int(step.keep)]

    def attend(self, cmd: Command, step: Step, slots: Slots, rows: Buffer, qkv: Buffer, weights: Weights,
               states: States, out: Buffer) -> None:
        """out [tokens][v_heads * dv] from the convolution's rows and the product's."""
        k = 4 * self.k_heads * self.dk
        z = 4 * self.channels
        b = z + 4 * self.out_width
        with _undone(slots, step):
            encode(cmd, "attn_linear",
                   [qkv, qkv, qkv, rows, rows, weights.a_log, weights.dt_bias, rows, weights.norm, *step.buffers, states.heads, out],
                   self.attend_params(step, slots), [0, k, 2 * k, b + 4 * self.v_heads, b, 0, 0, z, 0, 0, 0, 0, 0])


class Draws:
    """How a token is drawn from each of some rows of logits: numbers, or one a
    row. Temperature 0 takes the greatest; top_k 0, top_p 1 and min_p 0 keep all."""

    def __init__(self, gpu: Gpu, rows: int, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0):
        def column(value, kind):
            return gpu.upload_bytes(np.ascontiguousarray(np.broadcast_to(np.asarray(value, kind), rows)))

        self.rows = rows
        self.settings = (column(temperature, np.float32), column(top_k, np.uint32), column(top_p, np.float32),
                         column(min_p, np.float32))
        self.numbers = gpu.alloc_f32(rows)

    def sample(self, cmd: Command, logits: Buffer, vocab: int, tokens: Buffer, probs: Buffer,
               numbers: Optional[np.ndarray] = None) -> None:
        """tokens u32 [rows] and their probabilities from logits [rows][vocab]
        and one number from 0 to 1 a row (zeros until some are given). No command
        that draws may be under way when numbers are given."""
        if numbers is not None:
            numbers = np.ascontiguousarray(numbers, np.float32)
            if numbers.shape != (self.rows,):
                raise ValueError(f"{self.rows} rows are drawn, each with one number")
            self.numbers.write(numbers)
        encode(cmd, "sample_logits", [logits, *self.settings, self.numbers, tokens, probs], [self.rows, vocab, vocab])
