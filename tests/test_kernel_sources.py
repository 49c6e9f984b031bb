"""What the compiler has to be told about the inline assembly of the kernels, read from their sources."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "torch-convnd_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".h"))


def statements(text):
    """The operands of each inline assembly statement, up to its closing parenthesis."""
    for start in re.finditer(r"\basm(?:\s+volatile)?\s*\(", text):
        at, depth = start.end(), 1
        while depth:
            quoted = re.compile(r'"(?:[^"\\]|\\.)*"').match(text, at)
            if quoted:
                at = quoted.end()
                continue
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        yield text[start.end() : at - 1]


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_registers_written_by_name_are_clobbers(source):
    for statement in statements(source.read_text()):
        template = re.match(r'\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', statement)
        written = re.findall(r"\bs_mov_b32 (m0|vcc_lo|vcc_hi|s\d+),", template.group(1))
        clobbers = re.findall(r'"([^"]*)"', statement[template.end() :].rsplit(":", 1)[-1])
        for register in written:
            assert register in clobbers, f"{source.name}: {register} is written and not named: {statement}"
