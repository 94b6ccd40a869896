"""Rules of the gfx950 sources that a compiler does not check: it does not look inside assembly strings."""

from __future__ import annotations

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jitengine_amd", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.hpp")))


def _asm_strings(path: str) -> list:
    """The instructions of each assembly statement of a source."""
    text = open(path).read()
    return [re.split(r"\\n(?:\\t)?", "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', m)))
            for m in re.findall(r'asm volatile\(((?:\s*"(?:[^"\\]|\\.)*")+)', text)]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_a_wait_state_stands_between_m0_and_a_direct_load(path):
    """A load straight into LDS takes its LDS address from M0, one wait state after a scalar write of it at the
    earliest."""
    for code in _asm_strings(path):
        for i, ins in enumerate(code):
            if re.match(r"(global|buffer)_load_(lds_)?\w+", ins) and re.search(r"\blds\b|_lds_", ins):
                before = [c for c in code[:i] if c.strip()]
                assert len(before) >= 2 and before[-2].startswith("s_mov_b32 m0,") and before[-1].startswith("s_nop "), code


def test_the_direct_loads_are_found():
    found = {os.path.basename(p) for p in SOURCES if any("_lds_" in ins for code in _asm_strings(p) for ins in code)}
    assert found >= {"attention.hip", "kv8_attention.hip", "qmm_seg.hip", "probe.hip"}
