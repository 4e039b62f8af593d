"""Inline assembly leaves m0 to the compiler, which keeps values of its own there
(indirect register moves, some LDS accesses) and may hold one over several
uses: it takes m0 as an operand and never writes it."""
from __future__ import annotations

import re

import pytest

from turbinator_c_amd import build

SOURCES = sorted(p for end in ("hip", "h") for p in build.CSRC.glob(f"*.{end}"))
TEXT = r'"(?:[^"\\]|\\.)*"'


def statements(source: str):
    """Each statement's template and what follows it."""
    for found in re.finditer(rf"\basm\s+(?:volatile\s*)?\(((?:\s*{TEXT})+)((?:{TEXT}|[^;\"])*);",
                             source):
        yield "".join(t[1:-1] for t in re.findall(TEXT, found[1])), found[2]


def wrong(source: str) -> list[str]:
    """Templates that write m0, or that load into LDS without naming its place."""
    return [template for template, rest in statements(source)
            if re.search(r"\b[sv]_\w+\s+m0\b", template) or
            ("_load_lds_" in template and '"{m0}"' not in rest)]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_m0(path):
    assert not wrong(path.read_text())


def test_the_search_finds_statements():
    assert wrong(r'asm volatile("s_mov_b32 m0, %0\n\t" "s_nop 0" :: "s"(to) : "memory");')
    assert wrong('asm volatile("global_load_lds_dword %0, off" ::"v"(p) : "memory");')
    assert not wrong('asm volatile("global_load_lds_dword %1, off" ::"{m0}"(to), "v"(p));')
    assert not wrong('asm volatile("v_mov_b32 %0, m0" : "=v"(x));')
    found = {p.name: len(list(statements(p.read_text()))) for p in SOURCES}
    assert found["int8.hip"] == 3 and found["onboard.hip"] >= 7
