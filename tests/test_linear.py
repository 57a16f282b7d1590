"""Slots of qmr.linear, and the parameter words it makes (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

import qmr
from qmr import linear


def test_slots_are_fresh_until_tokens_are_kept():
    slots = linear.Slots(3)
    a, b = slots.open(), slots.open()
    assert slots.free == 1
    step = slots.step([(a, 5), (b, 0)])
    assert step.starts.tolist() == [0, 5, 5] and step.words.tolist() == [linear.FRESH, linear.FRESH | 1]
    assert step.tokens == 5 and step.most == 5
    # b had no token yet, and tokens that are not kept leave no state.
    assert slots.step([(b, 2)], keep=False).words.tolist() == [linear.FRESH | 1]
    step = slots.step([(b, 1), (a, 1)])
    assert step.words.tolist() == [linear.FRESH | 1, 0] and step.most == 1
    assert step.starts.dtype == np.uint32 and step.words.dtype == np.uint32
    assert slots.step([(b, 1)]).words.tolist() == [1]


def test_a_slot_that_is_taken_again_is_fresh():
    slots = linear.Slots(1)
    a = slots.open()
    slots.step([(a, 1)])
    with pytest.raises(MemoryError):
        slots.open()
    slots.close(a)
    b = slots.open()
    assert b != a and slots.step([(b, 1)]).words.tolist() == [linear.FRESH]
    with pytest.raises(KeyError):
        slots.step([(a, 1)])
    with pytest.raises(KeyError):
        slots.close(a)


def test_refusals():
    slots = linear.Slots(2)
    a = slots.open()
    for new in ([], [(a, 1), (a, 1)], [(a, -1)]):
        with pytest.raises(ValueError):
            slots.step(new)
    assert slots.step([(a, 1)]).words.tolist() == [linear.FRESH]  # nothing had changed
    for bad in (0, linear.FRESH):
        with pytest.raises(ValueError):
            linear.Slots(bad)


def test_words_fit_the_layouts():
    slots = linear.Slots(4)
    a, b = slots.open(), slots.open()
    step = slots.step([(a, 9), (b, 2)])
    layer = linear.Layer(2, 6, 32, 64, width=3, bias=True)
    assert layer.channels == 512 and layer.row == 512 + 384 + 12 and layer.out_width == 384
    sizes, _ = qmr.dispatch_layout("conv_causal", layer.convolve_params(step, slots))
    assert sizes == [4 * (10 * 908 + 512), 4 * 512 * 3, 4 * 512, 12, 8, 4 * 4 * 2 * 512, 4 * 11 * 512]
    sizes, _ = qmr.dispatch_layout("attn_linear", layer.attend_params(step, slots))
    assert sizes[3:9] == [4 * (10 * 908 + 6)] * 2 + [24, 24, 4 * (10 * 908 + 384), 256]
    assert sizes[9:] == [12, 8, 4 * 4 * 6 * 32 * 64, 4 * 11 * 384]
    assert layer.attend_params(step, slots)[13] == 9
    assert layer.attend_params(step, slots)[-1] == layer.convolve_params(step, slots)[-1] == 1
    step = slots.step([(a, 3)], keep=False)
    assert layer.attend_params(step, slots)[-1] == layer.convolve_params(step, slots)[-1] == 0
