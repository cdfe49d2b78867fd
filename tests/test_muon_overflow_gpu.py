"""The loss scaler's overflow test over Muon's matrices."""

from __future__ import annotations

import pytest
import torch

from minidist.optim import Muon

pytestmark = pytest.mark.gpu


def _optimizer():
    mats = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((40, 24), (1, 7), (300, 70), (40, 24))]
    vec = torch.nn.Parameter(torch.randn(10, device="cuda"))
    for p in (*mats, vec):
        p.grad = torch.ones_like(p)
    return Muon([dict(params=mats), dict(params=[vec])]), mats, vec


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_every_matrix_is_looked_at(value):
    opt, mats, vec = _optimizer()
    flag = torch.zeros(1, device="cuda")
    opt.check_nonfinite(flag)
    assert flag.item() == 0.0 and not any(opt.state[p] for p in mats)  # no moments are made for it
    for p in (*mats, vec):
        p.grad.view(-1)[-1] = value
        opt.check_nonfinite(flag)
        assert flag.item() == 1.0
        p.grad = torch.ones_like(p)  # elsewhere in memory
        flag.zero_()
        opt.check_nonfinite(flag)
        assert flag.item() == 0.0
    mats[0].grad = torch.ones(24, 40, device="cuda").t()
    mats[1].grad = torch.full((1, 7), value, device="cuda")
    opt.check_nonfinite(flag)
    assert flag.item() == 1.0


def test_one_launch_for_a_group():
    """As for AdamW's groups: one pass over all gradients of a group, no operation per matrix."""
    opt, _, _ = _optimizer()
    flag = torch.zeros(1, device="cuda")
    opt.check_nonfinite(flag)
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        opt.check_nonfinite(flag)
        torch.cuda.synchronize()
    kernels = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA]
    assert len(kernels) == 2 and all("nonfinite" in k for k in kernels), kernels
