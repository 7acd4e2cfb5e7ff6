"""CPU checks of the kernels' sources that no run can see today."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flashrwkv_amd" / "csrc"
SOURCES = sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")])
# An asm statement's template: the string literals before its first colon.
ASM = re.compile(r"\basm\s+volatile\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)")


def _blocks(text):
    for match in ASM.finditer(text):
        literals = re.findall(r"\"((?:[^\"\\]|\\.)*)\"", match.group(1))
        lines = "".join(literals).replace("\\t", " ").split("\\n")
        yield [line.strip() for line in lines if line.strip()]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_assembly_that_writes_m0_gives_its_value_back(path):
    """m0 cannot be declared as written, and the compiler may keep a value there: a
    block that writes it saves it first and restores it last (or takes what it needs
    there as an operand)."""
    for lines in _blocks(path.read_text()):
        if not any(re.match(r"s_\w+ m0,", line) for line in lines):
            continue
        saved = re.fullmatch(r"s_mov_b32 (%\d+), m0", lines[0])
        assert saved, lines
        assert lines[-1] == f"s_mov_b32 m0, {saved.group(1)}", lines


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_loads_to_lds_wait_for_m0(path):
    """One wait state between a write of m0 and a load to LDS, which the compiler
    keeps by itself and assembly has to."""
    for lines in _blocks(path.read_text()):
        # An operand in m0 is written right before the block.
        for before, line in zip(["s_mov_b32 m0, operand", *lines], lines):
            if line.endswith(" lds"):
                assert not re.match(r"s_\w+ m0,", before), lines


def test_the_scan_finds_blocks_and_would_see_a_lost_value():
    blocks = [b for p in SOURCES for b in _blocks(p.read_text())]
    assert any("m0" in line for b in blocks for line in b)
    assert sum(any(line.endswith(" lds") for line in b) for b in blocks) >= 2
    planted = list(_blocks('asm volatile("s_mov_b32 m0, %1\\n\\t" "s_nop 0" : : "s"(x));'))
    assert planted == [["s_mov_b32 m0, %1", "s_nop 0"]]
