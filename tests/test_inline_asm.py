"""Inline assembly of the kernels: what it writes without naming it as an output
has to stand among its clobbers, or the compiler keeps its own values there."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qwen-mlx-runner_amd" / "csrc"
SOURCES = sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.hpp")])
# Registers that an instruction's first operand names outright.
WRITES = re.compile(r'(?:"|\\n|\\t|;)\s*[sv]_\w+\s+(m0|vcc(?:_lo|_hi)?|exec(?:_lo|_hi)?|[sv]\d+|a\d+)\s*,')


def statements(text: str) -> list[str]:
    """The parts in brackets of every asm statement."""
    out = []
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, at, quoted = 1, m.end(), False
        while depth:
            c = text[at]
            if c == '"' and text[at - 1] != "\\":
                quoted = not quoted
            depth += 0 if quoted else (c == "(") - (c == ")")
            at += 1
        out.append(text[m.end():at - 1])
    return out


def unnamed(statement: str) -> set[str]:
    body = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', statement).group(1)
    rest = statement[len(body):]
    return {r for r in WRITES.findall(body) if f'"{r}"' not in rest}


def test_the_search_finds_a_missing_clobber():
    lost = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 4" : : "s"(to) : "memory");'
    assert [unnamed(s) for s in statements(lost)] == [{"m0"}]
    assert [unnamed(s) for s in statements(lost.replace('"memory"', '"memory", "m0"'))] == [set()]


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_registers_written_by_name_are_clobbers(source):
    for s in statements(source.read_text()):
        assert not unnamed(s), s
