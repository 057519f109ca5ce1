"""What the sources of the microscaled (MX) kernels have to state themselves, whatever the compiler makes of them today."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "ditserve_amd" / "csrc"
SOURCES = sorted(CSRC.glob("mx_*.hip"))


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_barriers_wait_for_lds_reads(path):
    """Behind a barrier LDS is filled anew: each wave states, right before it, that its own reads have landed."""
    text = path.read_text()
    for at in re.finditer(r"__builtin_amdgcn_s_barrier\(\)", text):
        last = text[:at.start()].rsplit("asm volatile(", 1)[1]
        assert "lgkmcnt(0)" in last and last.count(";") == 1, f"{path.name}:{text.count(chr(10), 0, at.start()) + 1}"


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_assembly_declares_m0(path):
    """Assembly that sets m0 (the LDS address of a DMA), in place or in an included body, says so to the compiler."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    for at in re.finditer(r"asm volatile\(", text):
        depth, end = 1, at.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        body = text[at.end():end]
        code = body + "".join((CSRC / name).read_text() for name in re.findall(r'#include "(\w+\.inc)"', body))
        if re.search(r"\bs_\w+ m0,", code):
            assert '"m0"' in body, f"{path.name}:{text.count(chr(10), 0, at.start()) + 1}"
