"""The status word that every kernel reports into, made by whatever call comes first."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST_CALL_IN_INFERENCE_MODE = """
import torch
import minidist as md
from minidist.ops import _native as nat

q = torch.randn(1, 3, 2, 16, device="cuda")
table = md.rotary_table(8, 10, device="cuda")
with torch.inference_mode():
    md.apply_rotary(q, None, table)
md.apply_rotary(q, None, table, torch.tensor([0, 10, -1], device="cuda"))
for expected in (True, False):  # reported once, then cleared
    try:
        nat.check_status()
    except nat.NativeError:
        assert expected
    else:
        assert not expected
print("cleared")
"""


@pytest.mark.gpu
def test_made_in_inference_mode_and_cleared_outside():
    proc = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_INFERENCE_MODE], capture_output=True, text=True,
                          timeout=120, cwd=ROOT)
    assert proc.returncode == 0 and "cleared" in proc.stdout, proc.stderr[-2000:]
