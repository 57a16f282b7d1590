"""The served attention block of examples/paged_attention.py, end to end."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

from qmr import paged

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "paged_attention", Path(__file__).resolve().parent.parent / "examples" / "paged_attention.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)

# The oracle rounds its keys and values from 64 bits, the kernel its own from
# 32: a value on the edge of two bf16 numbers may go to the other, 2^-8 of it
# at most. Keys and queries are normalised (elements to 4 * 1.5), so that moves
# a score by at most 36 * 2^-8 / sqrt(128) = 1.2e-2, and an output by as much
# where that key has all the weight. Mixed pages or positions are off by 0.1 to 1.
BOUND = 1.5e-2


@pytest.mark.parametrize("heads, kv_heads, dim, rotary, prompts, chunk, page", [
    (8, 2, 128, 128, [130, 33, 1], 50, 32),
    (4, 4, 64, 32, [20, 64, 7, 2], 64, 64),
])
def test_served_block(gpu, heads, kv_heads, dim, rotary, prompts, chunk, page):
    layer = paged.Attention(heads, kv_heads, dim, rotary, (rotary // 2,), eps=1e-6)
    lines = []
    worst = example.serve(gpu, layer, 512, prompts, chunk, 4, page, lines.append)
    assert len(lines) >= 4 + len(prompts)
    assert worst < BOUND
