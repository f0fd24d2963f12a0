"""Inline assembly in the kernels names the registers it writes beside its operands (CPU: the sources alone)."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCES = sorted((Path(__file__).resolve().parents[1] / "fast-attnres_amd" / "csrc").glob("*.h*"))


def _statements(text: str) -> list[str]:
    """The text of every asm statement, comments left out."""
    text = re.sub(r"//[^\n]*", "", text)
    return [text[m.start():text.index(";\n", m.start())] for m in re.finditer(r"\basm\b", text)]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_written_special_registers_are_clobbers(path):
    for statement in _statements(path.read_text()):
        template = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statement.split(":")[0]))
        clobbers = statement.split(":")[-1] if statement.count(":") >= 3 else ""
        for register in re.findall(r"\bs_\w+\s+(m0|vcc|exec|scc)\b", template):
            assert f'"{register}"' in clobbers, statement


def test_statements_are_found():
    found = [s for path in SOURCES for s in _statements(path.read_text())]
    assert any("m0" in s for s in found) and any("s_waitcnt" in s for s in found)
