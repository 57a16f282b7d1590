"""Page bookkeeping of qmr.paged, and the parameter words it makes (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

import qmr
from qmr import paged


def held(pages):
    return [p for ps in pages._held.values() for p in ps]


def test_steps_take_pages_as_lengths_grow():
    pages = paged.Pages(32, 8, 4)
    a, b = pages.open(), pages.open()
    step = pages.step([(a, 33), (b, 1)])
    assert step.starts.tolist() == [0, 33, 34] and step.lengths.tolist() == [33, 1]
    assert step.positions.tolist() == [*range(33), 0] and step.tokens == 34 and step.max_keys == 33
    assert pages.free == 5
    assert (step.table[0, 2:] == paged.NO_PAGE).all() and (step.table[1, 1:] == paged.NO_PAGE).all()
    assert len(set(held(pages))) == 3
    # The rest of the pages' positions come without new pages, in the step's order.
    step = pages.step([(b, 31), (a, 31)])
    assert pages.free == 5 and step.lengths.tolist() == [32, 64]
    assert step.positions.tolist() == [*range(1, 32), *range(33, 64)]
    step = pages.step([(a, 0)])
    assert step.tokens == 0 and step.lengths.tolist() == [64] and step.positions.dtype == np.int32


def test_close_and_trim_give_pages_back():
    pages = paged.Pages(32, 4, 4)
    a, b = pages.open(), pages.open()
    pages.step([(a, 64), (b, 40)])
    assert pages.free == 0
    pages.trim(a, 33)
    assert pages.free == 0 and pages.length(a) == 33
    pages.trim(a, 32)
    assert pages.free == 1
    pages.close(b)
    assert pages.free == 3
    with pytest.raises(KeyError):
        pages.length(b)
    c = pages.open()
    assert c not in (a, b)
    pages.step([(c, 96)])
    assert pages.free == 0 and len(set(held(pages))) == 4
    with pytest.raises(ValueError):
        pages.trim(a, 33)


@pytest.mark.parametrize("new, error", [
    ([(0, 65), (1, 64)], MemoryError),   # five pages of four
    ([(0, 97)], ValueError),             # past a sequence's columns
    ([(0, 1), (0, 1)], ValueError),
    ([(0, -1)], ValueError),
    ([(7, 1)], KeyError),
])
def test_a_step_that_cannot_be_changes_nothing(new, error):
    pages = paged.Pages(32, 4, 3)
    a, b = pages.open(), pages.open()
    assert (a, b) == (0, 1)
    with pytest.raises(error):
        pages.step(new)
    assert pages.free == 4 and pages.length(a) == pages.length(b) == 0 and held(pages) == []


@pytest.mark.parametrize("kind, sections, dealt", [("bf16", (32,), False), ("f16", (8, 12, 12), False), ("bf16", (12, 10, 10), True)])
def test_parameter_words_are_what_the_library_takes(kind, sections, dealt):
    pages = paged.Pages(64, 16, 8)
    seqs = [pages.open() for _ in range(3)]
    step = pages.step([(s, n) for s, n in zip(seqs, (70, 1, 5))])
    layer = paged.Attention(8, 2, 128, 64, sections, kind, dealt=dealt, eps=1e-6, window=40)
    sizes, _ = qmr.dispatch_layout("kv_append_rope_" + kind, layer.append_params(step, pages))
    row = 4 * layer.width
    assert sizes[0] == 75 * row + 4 * 8 * 128   # queries: the last token's heads end them
    assert sizes[1] == sizes[2] == 75 * row + 4 * 2 * 128
    cache = 2 * 16 * 2 * 64 * 128
    assert [s for s in sizes].count(cache) == 2
    sizes, _ = qmr.dispatch_layout("attn_paged_" + kind, layer.attend_params(step, pages))
    assert sizes[1:] == [16, 12, 96, cache, cache, 76 * 4 * 8 * 128]
