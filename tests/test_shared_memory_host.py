"""Dynamic shared memory that a kernel reads or writes more than four bytes at a time says how it is aligned: static arrays may
lie before it, and without a word the language promises its elements' alignment alone."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "musa-aiter_b200" / "csrc"
DECLARED = re.compile(r"extern\s+__shared__\s+(?:__align__\((\d+)\)\s+)?(?:unsigned\s+)?\w+\s+(\w+)\s*\[\]")


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.cu")), ids=lambda p: p.name)
def test_dynamic_shared_memory_is_aligned(path):
    text = path.read_text()
    assert text.count("extern __shared__") == len(DECLARED.findall(text))
    for align, name in DECLARED.findall(text):
        wide = re.search(rf"reinterpret_cast<(?:int4|uint4|float4|int64_t|uint64_t)\*>\({name}\b", text)
        assert align or not wide, f"{name} is used {wide.group(0)} and has no alignment of its own"
        assert not align or int(align) >= 16
