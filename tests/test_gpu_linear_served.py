"""The served linear-attention block of examples/linear_attention.py, end to end."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest

import qmr
from qmr import linear

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "linear_attention", Path(__file__).resolve().parent.parent / "examples" / "linear_attention.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)

# Both sides start from the same rows. A chunk leaves at most 400 roundings of
# 2^-24 of what its tokens bring, 2.4e-5, and the states forget; the output norm
# divides by a head's own rms, which makes that up to sqrt(dv) = 11 times the
# head's outputs at worst. Mixed slots, rows or gates are off by 0.1 to 1.
BOUND = 1e-3
# Weights are whole numbers of 2^-49 of the largest and sums exact; numpy's sum
# of a thousand weights in 64 bits rounds to 1e-13.
DRAW = 1e-10


@pytest.mark.parametrize("layer, hidden, vocab, prompts, chunk", [
    (linear.Layer(4, 8, 64, 64), 512, 1024, [130, 33, 1], 50),
    (linear.Layer(2, 6, 128, 32, width=3), 256, 9216, [20, 64, 7, 2], 64),
])
def test_served_block(gpu, layer, hidden, vocab, prompts, chunk):
    lines = []
    worst, missed = example.serve(gpu, layer, hidden, vocab, prompts, chunk, 4, lines.append)
    assert len(lines) >= 4 + len(prompts)
    assert worst < BOUND and missed < DRAW


def test_two_handles_at_once(gpu):
    """Two devices' handles, each with its stream and workspace, enqueue their
    steps before either waits; both get what each gets alone."""
    from linear_cases import Linear
    from sample_cases import Sample

    cases = [(Linear([300, 40, 1], 2, 4, 64, 64, seed=s), Sample(np.random.default_rng(s).standard_normal((3, 70001)), 0.7, 50, 0.9))
             for s in range(2)]
    alone = [(case.run(gpu), draw.run(gpu)) for case, draw in cases]
    handles = [qmr.Gpu("aligned") for _ in cases]
    try:
        for _ in range(3):
            pending = []
            for g, (case, draw) in zip(handles, cases):
                up = g.upload_bytes
                rows = [up(x) for x in (case.q, case.k, case.v, case.a, case.b, case.a_log, case.dt_bias, case.z, case.norm,
                                        case.starts, case.slots, case.state)]
                out = g.alloc_f32(case.tokens * case.v_heads * case.dv)
                small = [up(draw.logits), *(up(x) for x in (draw.temperature, draw.k, draw.p, draw.min_p, draw.u))]
                tokens, probs = g.alloc(12), g.alloc(12)
                cmd = g.begin()
                kw, vw, h = case.k_heads * case.dk, case.v_heads * case.dv, case.v_heads
                words = case.params([kw, kw, vw, h, h, vw, vw])
                # The draw's workspace is that of the attention before and after it.
                for _ in range(2):
                    cmd.encode("sample_logits", [*small, tokens, probs], [3, 70001, 70001], 3 * 1024, 64)
                    cmd.encode("attn_linear", [*rows, out], words, qmr.dispatch_layout("attn_linear", words)[1], 64)
                    words[-1] = 0
                pending.append((cmd, rows[-1], out, tokens, probs))
            for g, (case, _), ((want, state), (want_tokens, want_probs)), (cmd, after, out, tokens, probs) in zip(
                    handles, cases, alone, pending):
                cmd.finish()
                cmd.release()
                assert np.array_equal(after.read(np.float32, state.size).reshape(state.shape), state)
                assert np.array_equal(tokens.read(np.uint32, 3), want_tokens)
                assert np.array_equal(probs.read(np.float32, 3), want_probs)
                assert np.isfinite(out.read(np.float32, want.size)).all()
    finally:
        for g in handles:
            g.close()
