"""The sources order their asynchronous copies for the compiler: an ``asm`` statement that starts, commits or
waits for a cp.async reads or writes memory that its operands do not name, so it has to say "memory"; a plain read of
shared memory behind the wait could otherwise be moved in front of it."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "sophia_b200" / "csrc"
STATEMENT = re.compile(r"asm\s+volatile\s*\((?:[^()\"]|\"(?:[^\"\\]|\\.)*\"|\((?:[^()]|\([^()]*\))*\))*\)", re.S)


@pytest.mark.parametrize("path", sorted(p for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh", ".h")),
                         ids=lambda p: p.name)
def test_copies_name_memory(path):
    text = path.read_text()
    found = [m.group(0) for m in STATEMENT.finditer(text) if "cp.async" in m.group(0)]
    named = re.compile(r"\"\{?\s*cp\.async[^\"\n]*\"")
    assert sum(len(named.findall(s)) for s in found) == len(named.findall(text))  # none that the pattern misses
    for s in found:
        assert '"memory"' in s, s
