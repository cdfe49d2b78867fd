"""Kernels whose loops must not go through local memory, by what the assembler said when it built them."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

OBJ = Path(__file__).resolve().parent.parent / "minidist" / "_lib" / "obj"


@pytest.mark.parametrize("source,kernel,most", [("logprobs", "forward_kernel", 32), ("logprobs", "backward_kernel", 0),
                                                ("rotary", "rotary_kernel", 0), ("muon", "product_kernel", 0)])
def test_spills(source, kernel, most):
    """``most`` bytes: what a few values kept across the loops take, not a loop's own."""
    log = OBJ / f"{source}.ptxas.txt"
    if not log.exists():
        pytest.skip("not built here")
    found = re.findall(r"Function properties for (\S+)\n\s+\d+ bytes stack frame, (\d+) bytes spill stores", log.read_text())
    spills = {name: int(n) for name, n in found if kernel in name}
    assert spills and max(spills.values()) <= most, {k: v for k, v in spills.items() if v > most}
