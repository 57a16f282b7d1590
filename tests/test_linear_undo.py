"""Steps of qmr.linear that were refused (no GPU)."""
from __future__ import annotations

import pytest

import qmr
from qmr import linear


class Refusing:
    """A command that refuses dispatches of one name, and counts the others."""

    def __init__(self, name: str):
        self.name, self.taken = name, 0

    def encode(self, name, *rest, **more):
        if name == self.name:
            raise qmr.QmrError(1, "refused")
        self.taken += 1


LAYER = linear.Layer(1, 2, 32, 32)


def run(cmd, step, slots):
    weights, states = linear.Weights(*[None] * 3), linear.States(None, None)
    LAYER.convolve(cmd, step, slots, None, None, None, states, None)
    LAYER.attend(cmd, step, slots, None, None, weights, states, None)


@pytest.mark.parametrize("name", ["conv_causal", "attn_linear"])
def test_a_refused_step_leaves_its_sequences_fresh(name):
    """Their slots hold what the last owner left, or what a layer before the
    refusal made of them: neither may be read."""
    slots = linear.Slots(3)
    old, new, idle = slots.open(), slots.open(), slots.open()
    run(Refusing(""), slots.step([(old, 3)]), slots)
    step = slots.step([(new, 2), (old, 1), (idle, 0)])
    assert step.words.tolist() == [1 | linear.FRESH, 0, 2 | linear.FRESH]
    with pytest.raises(qmr.QmrError, match="refused"):
        run(Refusing(name), step, slots)
    again = slots.step([(new, 2), (old, 1), (idle, 0)])
    assert again.words.tolist() == step.words.tolist()
    cmd = Refusing("")
    run(cmd, again, slots)
    assert cmd.taken == 2
    assert slots.step([(new, 1), (old, 1), (idle, 1)]).words.tolist() == [1, 0, 2 | linear.FRESH]


def test_undo_after_a_failure_elsewhere():
    slots = linear.Slots(2)
    a, b = slots.open(), slots.open()
    first = slots.step([(a, 4)])
    slots.undo(first)
    slots.undo(first)  # once is all
    second = slots.step([(a, 4), (b, 1)])
    assert second.words.tolist() == [linear.FRESH, 1 | linear.FRESH]
    third = slots.step([(a, 1)])
    # What a later step has gone on from took place.
    slots.undo(first)
    slots.undo(second)
    assert slots.step([(a, 1), (b, 1)]).words.tolist() == [0, 1 | linear.FRESH]
    slots.undo(third)
    assert slots.step([(a, 1)]).words.tolist() == [0]


def test_undo_of_steps_that_keep_nothing_and_of_closed_sequences():
    slots = linear.Slots(1)
    a = slots.open()
    step = slots.step([(a, 2)], keep=False)
    slots.undo(step)
    assert slots.step([(a, 2)], keep=False).words.tolist() == [linear.FRESH]
    kept = slots.step([(a, 2)])
    slots.undo(slots.step([(a, 3)], keep=False))  # tried, and not kept: the step before stands
    assert slots.step([(a, 1)], keep=False).words.tolist() == [0]
    slots.close(a)
    b = slots.open()
    slots.undo(kept)
    assert slots.step([(b, 1)]).words.tolist() == [linear.FRESH]
    with pytest.raises(KeyError):
        slots.step([(a, 1)])
