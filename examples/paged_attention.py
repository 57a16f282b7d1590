"""The attention block of one decoder layer, served: prompts in chunks, then
tokens of all sequences together, with a sequence that comes and one that goes.

    python examples/paged_attention.py [--tokens N]

Packed Q4 products make queries, keys and values side by side and take the
heads' outputs back; between them stand the append to the paged cache and the
attention over it. The weights are synthetic. Every step's attention is checked
against numpy in 64 bits over the keys and values that the products gave.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "qwen-mlx-runner_amd"))

import qmr
from qmr import paged, synth


class Block:
    """Products, norms and cache of one layer."""

    def __init__(self, gpu: qmr.Gpu, layer: paged.Attention, hidden: int, pages: paged.Pages, most_tokens: int):
        self.gpu, self.layer, self.hidden, self.pages = gpu, layer, hidden, pages
        self.in_w = self._matrix(layer.width, hidden, "in")
        self.out_w = self._matrix(hidden, layer.heads * layer.dim, "out")
        rng = np.random.default_rng(5)
        self.norms = [rng.uniform(0.5, 1.5, layer.dim).astype(np.float32) for _ in range(2)]
        self.norm_buffers = [gpu.upload_f32(n) for n in self.norms]
        self.freqs = (1e6 ** (-np.arange(layer.rotary // 2) / (layer.rotary // 2))).astype(np.float32)
        self.freq_buffer = gpu.upload_f32(self.freqs)
        self.cache = layer.cache(gpu, pages)
        self.qkv = gpu.alloc_f32(most_tokens * layer.width)
        self.heads_out = gpu.alloc_f32(most_tokens * layer.heads * layer.dim)
        self.y = gpu.alloc_f32(most_tokens * hidden)

    def _matrix(self, rows: int, cols: int, tag: str):
        m = synth.q4_bf16_matrix(rows, cols, synth.DEFAULT_SEED, tag)
        return [self.gpu.upload_bytes(a) for a in (m.w, m.s, m.b)], rows, cols

    def _product(self, cmd: qmr.Command, matrix, x: qmr.Buffer, y: qmr.Buffer, tokens: int) -> None:
        w, rows, cols = matrix
        name = "matmul_affine_bf16" if tokens <= 4 else "matmul_affine_wide_bf16"
        for at in range(0, tokens, 256):
            paged.encode(cmd, name, [*w, x, y], [rows, cols, 4, 64, min(256, tokens - at)],
                         [0, 0, 0, 4 * at * cols, 4 * at * rows])

    def step(self, new, x: np.ndarray):
        """One step of (sequence, tokens) over x [tokens][hidden]: the heads'
        outputs, the block's, the products' rows and the GPU's seconds."""
        step = self.pages.step(new).upload(self.gpu)
        # One axis here; a step with images gives a row of positions an axis.
        positions = self.gpu.upload_bytes(np.tile(step.positions, (len(self.layer.sections), 1)))
        xb = self.gpu.upload_f32(x)
        cmd = self.gpu.begin()
        self._product(cmd, self.in_w, xb, self.qkv, step.tokens)
        cmd.finish()
        rows = self.qkv.read(np.float32, step.tokens * self.layer.width).reshape(step.tokens, -1)
        cmd = self.gpu.begin()
        self.layer.append(cmd, step, self.pages, self.qkv, self.cache, positions, self.freq_buffer, *self.norm_buffers)
        self.layer.attend(cmd, step, self.pages, self.qkv, self.cache, self.heads_out)
        self._product(cmd, self.out_w, self.heads_out, self.y, step.tokens)
        seconds = cmd.finish().gpu_seconds
        width = self.layer.heads * self.layer.dim
        return (self.heads_out.read(np.float32, step.tokens * width).reshape(step.tokens, width),
                self.y.read(np.float32, step.tokens * self.hidden).reshape(step.tokens, self.hidden), rows, seconds)


class Plain:
    """The same attention in numpy, over its own unpaged keys and values: turned
    in 64 bits, kept as the cache keeps them."""

    def __init__(self, block: Block):
        self.block, self.keys, self.values = block, {}, {}

    def _turned(self, x, norm, positions):
        layer, half = self.block.layer, self.block.layer.rotary // 2
        x = x.astype(np.float64).reshape(len(positions), -1, layer.dim)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + layer.eps) * norm
        t = positions[:, None, None] * self.block.freqs.astype(np.float64)
        a, b = x[..., :half].copy(), x[..., half:2 * half].copy()
        x[..., :half], x[..., half:2 * half] = a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)
        return x

    @staticmethod
    def _kept(x):
        return synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(x.astype(np.float32))).astype(np.float64)

    def step(self, new, rows):
        layer, at, out = self.block.layer, 0, []
        h, kv, d = layer.heads, layer.kv_heads, layer.dim
        for seq, n in new:
            length = self.block.pages.length(seq)
            positions = np.arange(length - n, length)
            q, k, v = np.split(rows[at:at + n], [h * d, (h + kv) * d], axis=1)
            at += n
            q = self._turned(q, self.block.norms[0], positions)
            k = self._kept(self._turned(k, self.block.norms[1], positions))
            v = self._kept(v.reshape(n, kv, d))
            k = self.keys[seq] = np.concatenate([self.keys[seq][:length - n], k]) if seq in self.keys else k
            v = self.values[seq] = np.concatenate([self.values[seq][:length - n], v]) if seq in self.values else v
            s = np.einsum("thd,khd->htk", q, np.repeat(k, h // kv, axis=1)) * d ** -0.5
            s = np.where(np.arange(length) <= positions[:, None], s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out.append(np.einsum("htk,khd->thd", p, np.repeat(v, h // kv, axis=1)).reshape(n, h * d))
        return np.concatenate(out)


def serve(gpu: qmr.Gpu, layer: paged.Attention, hidden: int, prompts, chunk: int, tokens: int, page: int = 64,
          report=print):
    """Prompts in chunks, then `tokens` steps of one token of each sequence. In
    the middle the first sequence ends, another takes its pages, and the last
    one gives back two tokens that it wrote. The largest error of any step,
    relative to its largest output."""
    columns = -(-(max(prompts) + tokens + 1) // page)
    pages = paged.Pages(page, sum(-(-(p + tokens + 1) // page) for p in prompts), columns)
    block = Block(gpu, layer, hidden, pages, max(chunk, len(prompts)))
    plain, rng, worst = Plain(block), np.random.default_rng(7), 0.0

    def step(new):
        nonlocal worst
        got, y, rows, seconds = block.step(new, rng.standard_normal((sum(n for _, n in new), hidden)).astype(np.float32))
        want = plain.step(new, rows)
        off = float(np.abs(got - want).max() / np.abs(want).max())
        worst = max(worst, off)
        assert np.isfinite(y).all()
        report(f"{len(new)} sequences, {len(got):4d} tokens, {max(pages.length(s) for s, _ in new):6d} positions at most: "
               f"{seconds * 1e6:8.1f} us, off by {off:.1e}; {pages.free} pages left")

    def prompt(length):
        seq = pages.open()
        for at in range(0, length, chunk):
            step([(seq, min(chunk, length - at))])
        return seq

    seqs = [prompt(n) for n in prompts]
    for i in range(tokens):
        if i == tokens // 2:
            first = pages.length(seqs[0])
            pages.close(seqs.pop(0))
            seqs.append(prompt(max(1, first // 2)))
            pages.trim(seqs[-2], pages.length(seqs[-2]) - 2)
        step([(s, 1) for s in seqs])
    return worst


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=8, help="steps after the prompts")
    args = ap.parse_args()
    layer = paged.Attention(heads=24, kv_heads=4, dim=256, rotary=64, sections=(32,), eps=1e-6)
    with qmr.Gpu() as gpu:
        worst = serve(gpu, layer, 5120, [300, 77, 1], 256, args.tokens)
    print(f"largest error: {worst:.1e}")


if __name__ == "__main__":
    main()
