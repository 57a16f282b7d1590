"""Linear attention and draws on two device handles whose launches overlap."""
import numpy as np
import pytest

import qmr
from linear_cases import Linear
from sample_cases import Sample

pytestmark = pytest.mark.gpu

VOCAB = 70001


class Queued:
    """A command on a handle of its own: a draw, the attention that keeps its
    states, the draw again, and the attention from those states, all in one
    workspace. Buffers live as long as this does."""

    def __init__(self, seed: int):
        self.gpu = qmr.Gpu("aligned")
        self.case = Linear([300, 40, 1], 2, 4, 64, 64, seed=seed)
        self.draw = Sample(np.random.default_rng(seed).standard_normal((3, VOCAB)), 0.7, 50, 0.9, seed=seed)
        up, c, d = self.gpu.upload_bytes, self.case, self.draw
        self.rows = [up(x) for x in (c.q, c.k, c.v, c.a, c.b, c.a_log, c.dt_bias, c.z, c.norm, c.starts, c.slots, c.state)]
        self.settings = [up(x) for x in (d.logits, d.temperature, d.k, d.p, d.min_p, d.u)]
        self.out = [self.gpu.alloc_f32(c.tokens * c.v_heads * c.dv) for _ in range(2)]
        self.drawn = [(self.gpu.alloc(12), self.gpu.alloc(12)) for _ in range(2)]
        kw, vw, h = c.k_heads * c.dk, c.v_heads * c.dv, c.v_heads
        self.words = c.params([kw, kw, vw, h, h, vw, vw])
        self.threads = qmr.dispatch_layout("attn_linear", self.words)[1]

    def encode(self, hold: int):
        self.rows[-1].write(self.case.state)
        self.cmd = self.gpu.begin()
        self.cmd.delay(hold)
        for keep in (1, 0):
            self.words[-1] = keep
            self.cmd.encode("sample_logits", [*self.settings, *self.drawn[keep]], [3, VOCAB, VOCAB], 3 * 1024, 64)
            self.cmd.encode("attn_linear", [*self.rows, self.out[keep]], self.words, self.threads, 64)

    def finish(self):
        self.cmd.finish()
        self.cmd.release()
        return ([b.read(np.float32, self.case.tokens * self.case.v_heads * self.case.dv) for b in self.out],
                self.rows[-1].read(np.float32, self.case.state.size),
                [(t.read(np.uint32, 3), p.read(np.float32, 3)) for t, p in self.drawn])


def test_two_handles_whose_launches_are_queued_together(gpu):
    pair = [Queued(seed) for seed in range(2)]
    try:
        want = []
        for q in pair:
            first, state = q.case.run(gpu)
            tokens, probs = q.draw.run(gpu)
            q.case.state, before = state, q.case.state
            q.case.keep = False
            second, _ = q.case.run(gpu)
            q.case.state, q.case.keep = before, True
            want.append((second.ravel(), first.ravel(), state.ravel(), tokens, probs))
        for _ in range(4):  # the first grows the workspaces
            for q in pair:
                q.encode(3000)
            for q, (second, first, state, tokens, probs) in zip(pair, want):
                out, after, drawn = q.finish()
                assert np.array_equal(out[1], first) and np.array_equal(out[0], second)
                assert np.array_equal(after, state)
                for t, p in drawn:
                    assert np.array_equal(t, tokens) and np.array_equal(p, probs)
    finally:
        for q in pair:
            q.gpu.close()
