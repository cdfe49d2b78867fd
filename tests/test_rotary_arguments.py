"""Positions and tables of ``apply_rotary`` beside the common ones."""

from __future__ import annotations

import pytest
import torch

import minidist as md

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("bad", [-1, -8, 8, 2**40])
@pytest.mark.parametrize("grad", [False, True])
def test_position_outside_the_table_raises_on_cpu(bad, grad):
    q = torch.randn(2, 4, 2, 16, requires_grad=grad)
    table = md.rotary_table(16, 8)
    for pos in (torch.tensor([0, 1, bad, 7]), torch.tensor([[0, 1, 2, 3], [4, bad, 6, 7]])):
        with pytest.raises(IndexError):
            md.apply_rotary(q, None, table, pos)
    md.apply_rotary(q, None, table, torch.tensor([0, 7, 7, 0]))
    md.apply_rotary(q[:, :0], None, table, torch.zeros(0, dtype=torch.long))
