"""One linear-attention block with its head, served: prompts in chunks, then
drawn tokens of all sequences together, with a sequence that comes and one that
goes.

    python examples/linear_attention.py [--tokens N]

Packed Q4 products make a row of queries, keys, values and gates, take the
heads' outputs back and give the logits; between them stand the convolution,
the linear attention and the draw. The weights are synthetic. Every step is
checked against numpy in 64 bits: the heads' outputs over the rows that the
products gave, the tokens over the logits.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "qwen-mlx-runner_amd"))

import qmr
from qmr import linear, paged, synth


class Block:
    """Products, weights and states of one layer, and the head."""

    def __init__(self, gpu: qmr.Gpu, layer: linear.Layer, hidden: int, vocab: int, slots: linear.Slots, most_tokens: int):
        self.gpu, self.layer, self.hidden, self.vocab, self.slots = gpu, layer, hidden, vocab, slots
        self.in_w = self._matrix(layer.row, hidden, "in")
        self.out_w = self._matrix(hidden, layer.out_width, "out")
        self.head = self._matrix(vocab, hidden, "head")
        rng = np.random.default_rng(5)
        self.filters = rng.uniform(-0.5, 0.5, (layer.channels, layer.width)).astype(np.float32)
        self.a_log = np.log(rng.uniform(1, 16, layer.v_heads)).astype(np.float32)
        self.dt_bias = rng.uniform(-6, -2, layer.v_heads).astype(np.float32)
        self.norm = rng.uniform(0.5, 1.5, layer.dv).astype(np.float32)
        self.filter_buffer = gpu.upload_f32(self.filters)
        self.weights = linear.Weights(*(gpu.upload_f32(w) for w in (self.a_log, self.dt_bias, self.norm)))
        self.states = layer.states(gpu, slots)
        self.rows, self.qkv = gpu.alloc_f32(most_tokens * layer.row), gpu.alloc_f32(most_tokens * layer.channels)
        self.heads_out, self.y = gpu.alloc_f32(most_tokens * layer.out_width), gpu.alloc_f32(most_tokens * hidden)
        self.logits = gpu.alloc_f32(slots.slots * vocab)
        self.tokens, self.probs = gpu.alloc(4 * slots.slots), gpu.alloc_f32(slots.slots)

    def _matrix(self, rows: int, cols: int, tag: str):
        m = synth.q4_bf16_matrix(rows, cols, synth.DEFAULT_SEED, tag)
        return [self.gpu.upload_bytes(a) for a in (m.w, m.s, m.b)], rows, cols

    @staticmethod
    def _product(cmd: qmr.Command, matrix, x: qmr.Buffer, y: qmr.Buffer, tokens: int, x_row: int = 0, y_row: int = 0) -> None:
        w, rows, cols = matrix
        name = "matmul_affine_bf16" if tokens <= 4 else "matmul_affine_wide_bf16"
        for at in range(0, tokens, 256):
            paged.encode(cmd, name, [*w, x, y], [rows, cols, 4, 64, min(256, tokens - at)],
                         [0, 0, 0, 4 * (x_row + at) * cols, 4 * (y_row + at) * rows])

    def step(self, new, x: np.ndarray, draws: linear.Draws, numbers: np.ndarray, keep: bool = True):
        """One step of (sequence, tokens) over x [tokens][hidden], one command: a
        token drawn after each sequence's last one. The products' rows, the heads'
        outputs, the logits, the tokens and the GPU's seconds."""
        layer, slots = self.layer, self.slots
        step = slots.step(new, keep).upload(self.gpu)
        xb = self.gpu.upload_f32(x)
        cmd = self.gpu.begin()
        self._product(cmd, self.in_w, xb, self.rows, step.tokens)
        layer.convolve(cmd, step, slots, self.rows, self.filter_buffer, self.filter_buffer, self.states, self.qkv)
        layer.attend(cmd, step, slots, self.rows, self.qkv, self.weights, self.states, self.heads_out)
        self._product(cmd, self.out_w, self.heads_out, self.y, step.tokens)
        for s, end in enumerate(step.starts[1:]):
            self._product(cmd, self.head, self.y, self.logits, 1, int(end) - 1, s)
        draws.sample(cmd, self.logits, self.vocab, self.tokens, self.probs, numbers)
        seconds = cmd.finish().gpu_seconds
        read = lambda b, n, w: b.read(np.float32, n * w).reshape(n, w)
        return (read(self.rows, step.tokens, layer.row), read(self.heads_out, step.tokens, layer.out_width),
                read(self.logits, len(new), self.vocab), self.tokens.read(np.uint32, len(new)), seconds)


class Plain:
    """The same layer in numpy, token after token, over its own states."""

    def __init__(self, block: Block):
        self.block, self.inputs, self.heads = block, {}, {}

    def step(self, new, rows, keep=True):
        b, layer, at, out = self.block, self.block.layer, 0, []
        hk, hv, dk, dv = layer.k_heads, layer.v_heads, layer.dk, layer.dv
        sigmoid = lambda v: 1 / (1 + np.exp(-v))
        for seq, n in new:
            mine = rows[at:at + n].astype(np.float64)
            at += n
            before = self.inputs.get(seq, np.zeros((layer.width - 1, layer.channels)))
            S = self.heads.get(seq, np.zeros((hv, dk, dv)))
            x = np.concatenate([before, mine[:, :layer.channels]])
            for t, row in enumerate(mine):
                c = (x[t:t + layer.width].T * b.filters).sum(1)
                q, k, v = np.split(c * sigmoid(c), [hk * dk, 2 * hk * dk])
                q, k = (np.repeat(a / np.sqrt((a * a).sum(-1, keepdims=True) + layer.qk_eps), hv // hk, axis=0)
                        for a in (q.reshape(hk, dk), k.reshape(hk, dk)))
                z, beta, a = np.split(row[layer.channels:], [hv * dv, hv * dv + hv])
                S = np.exp(-np.exp(b.a_log) * np.logaddexp(0, a + b.dt_bias))[:, None, None] * S
                u = sigmoid(beta)[:, None] * (v.reshape(hv, dv) - np.einsum("hij,hi->hj", S, k))
                S = S + k[:, :, None] * u[:, None, :]
                o = np.einsum("hij,hi->hj", S, q) * dk ** -0.5
                z = z.reshape(hv, dv)
                out.append((o / np.sqrt((o * o).mean(-1, keepdims=True) + layer.out_eps) * b.norm * z * sigmoid(z)).ravel())
            if keep:
                self.inputs[seq], self.heads[seq] = x[len(mine):], S
        return np.array(out)

    @staticmethod
    def missed(logits, temperature, k, p, number, token):
        """By how much of the weight `number` lies outside the token's share."""
        order = np.argsort(-logits, kind="stable")[:k]
        w = np.exp((logits[order].astype(np.float64) - logits[order[0]]) / temperature)
        kept = order[:max(1, int((np.cumsum(w) - w < p * w.sum()).sum()))]
        by_index = np.sort(kept)
        if token not in by_index:
            return 1.0
        w = np.exp((logits[by_index].astype(np.float64) - logits[order[0]]) / temperature)
        up_to, at = np.cumsum(w) / w.sum(), int(np.searchsorted(by_index, token))
        return max(number - up_to[at], (up_to[at - 1] if at else 0.0) - number, 0.0)


def serve(gpu: qmr.Gpu, layer: linear.Layer, hidden: int, vocab: int, prompts, chunk: int, tokens: int, report=print):
    """Prompts in chunks, then `tokens` steps of one drawn token of each
    sequence; in the middle the first sequence ends and another takes its slot,
    and three tokens of the last are tried and not kept. The largest error of a
    step, relative to its largest output, and the most that a draw missed by."""
    slots = linear.Slots(len(prompts))
    block = Block(gpu, layer, hidden, vocab, slots, max(chunk, len(prompts), 3))
    plain, rng, worst, missed = Plain(block), np.random.default_rng(7), 0.0, 0.0
    embed = rng.standard_normal((vocab, hidden)).astype(np.float32)
    temperature, k, p = 0.8, 40, 0.95

    def step(new, ids, keep=True):
        nonlocal worst, missed
        draws = linear.Draws(gpu, len(new), temperature, k, p)
        numbers = rng.random(len(new), np.float32)
        rows, got, logits, drawn, seconds = block.step(new, embed[ids], draws, numbers, keep)
        want = plain.step(new, rows, keep)
        off = float(np.abs(got - want).max() / np.abs(want).max())
        by = max(Plain.missed(x, temperature, k, p, float(u), t) for x, u, t in zip(logits, numbers, drawn))
        worst, missed = max(worst, off), max(missed, by)
        report(f"{len(new)} sequences, {len(got):4d} tokens: {seconds * 1e6:8.1f} us, off by {off:.1e}; drew {drawn.tolist()}")
        return drawn

    def prompt(length):
        seq, ids = slots.open(), rng.integers(0, vocab, length)
        for at in range(0, length, chunk):
            last = step([(seq, min(chunk, length - at))], ids[at:at + chunk])
        return seq, int(last[0])

    live = [prompt(n) for n in prompts]
    for i in range(tokens):
        if i == tokens // 2:
            slots.close(live.pop(0)[0])
            live.append(prompt(chunk // 2 + 1))
            step([(live[-1][0], 3)], rng.integers(0, vocab, 3), keep=False)
        drawn = step([(seq, 1) for seq, _ in live], [token for _, token in live])
        live = [(seq, int(token)) for (seq, _), token in zip(live, drawn)]
    return worst, missed


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=8, help="steps after the prompts")
    args = ap.parse_args()
    layer = linear.Layer(k_heads=16, v_heads=48, dk=128, dv=128)
    with qmr.Gpu() as gpu:
        worst, missed = serve(gpu, layer, 5120, 32000, [300, 77, 1], 256, args.tokens)
    print(f"largest error: {worst:.1e}; a draw missed by {missed:.1e} at most")


if __name__ == "__main__":
    main()
