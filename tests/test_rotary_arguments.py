"""Positions and tables of ``apply_rotary`` beside the common ones."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import rotary as R

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


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [2, 4, 6, 10, 12, 16, 50])
def test_table_that_starts_anywhere(device, dtype, interleaved, rotary):
    """Rows from an offset on (to continue a sequence), and a table inside another buffer."""
    q = torch.randn(2, 7, 3, 52, device=device).to(dtype)
    table = md.rotary_table(rotary, 20, device=device)
    for first in (1, 2, 3, 5):
        want = md.apply_rotary(q, None, table, torch.arange(first, first + 7, device=device), interleaved=interleaved)[0]
        assert torch.equal(md.apply_rotary(q, None, table[first:], interleaved=interleaved)[0], want)
        flat = torch.zeros(first + table.numel(), device=device)
        flat[first:] = table.flatten()
        inside = flat[first:].view(table.shape)
        assert torch.equal(md.apply_rotary(q, None, inside[first:], interleaved=interleaved)[0], want)
    if device == "cuda":
        nat.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_turning_in_place_is_a_change_that_autograd_sees(device):
    qkv = torch.randn(6, 3 * 2 * 16, device=device)
    w = torch.randn(6, 3 * 2 * 16, device=device, requires_grad=True)
    y = (w * qkv).sum()
    version = qkv._version
    R.rotate_packed_(qkv, 2, md.rotary_table(16, 3, device=device), batch=2)
    assert qkv._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("device", DEVICES)
def test_a_table_that_asks_for_a_gradient_is_refused(device):
    """It would get one or none depending on the device and on whether the queries ask for theirs."""
    table = md.rotary_table(16, 8, device=device).requires_grad_(True)
    for grad in (False, True):
        q = torch.randn(1, 4, 2, 16, device=device, requires_grad=grad)
        with pytest.raises(ValueError, match="gradient"):
            md.apply_rotary(q, None, table)
        with torch.no_grad():
            md.apply_rotary(q, None, table)


@pytest.mark.parametrize("bad", [dict(factor=float("inf")), dict(factor=float("nan")), dict(original_positions=0),
                                 dict(beta_slow=0.0), dict(beta_fast=0.5), dict(beta_fast=float("nan")),
                                 dict(beta_fast=float("inf"))])
def test_scaling_refusals(bad):
    """What would make a table of NaN, of nothing turning, or fail inside it."""
    with pytest.raises(ValueError, match="RotaryScaling"):
        md.RotaryScaling("yarn", **{"factor": 2.0, **bad})
    assert md.rotary_table(16, 8, scaling=md.RotaryScaling("yarn", 2.0, 1, beta_fast=2.0, beta_slow=2.0)).isfinite().all()
