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
