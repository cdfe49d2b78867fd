"""Gradients that do not lie as their parameters do, and copies that were stale, in FusedAdamW's kernels."""

from __future__ import annotations

import pytest
import torch

from minidist.models.fused_gpt import bf16_weight
from minidist.optim import FusedAdamW


@pytest.mark.gpu
def test_transposed_gradients():
    """Each is copied for the kernel; the copies have to live until it has run."""
    g = torch.Generator().manual_seed(0)
    values = [(torch.randn(64, 48, generator=g).cuda(), torch.randn(48, 64, generator=g).cuda()) for _ in range(6)]

    def run(order):
        params = [torch.nn.Parameter(w.clone()) for w, _ in values]
        opt = FusedAdamW(params, lr=0.1)
        for _ in range(2):
            for p, (_, t) in zip(params, values):
                p.grad = order(t.t())
            opt.step()
        return params

    for a, b in zip(run(lambda t: t), run(lambda t: t.contiguous())):
        assert torch.equal(a, b)
    params = [torch.nn.Parameter(w.clone()) for w, _ in values]
    opt, flag = FusedAdamW(params, lr=0.1), torch.zeros(1, device="cuda")
    for i, (p, (_, t)) in enumerate(zip(params, values)):
        p.grad = (t * (float("inf") if i == 0 else 1.0)).t()
    opt.check_nonfinite(flag)
    assert flag.item() == 1.0


@pytest.mark.gpu
def test_stale_copies_stay_stale():
    """Weights changed between backward and step: the step does not refresh their bf16 copies, and must
    not call them fresh."""
    params = [torch.nn.Parameter(torch.randn(32, 16, device="cuda")) for _ in range(3)]
    opt = FusedAdamW(params, lr=0.1)
    for p in params:
        bf16_weight(p)
        p.grad = torch.ones_like(p)
    with torch.no_grad():
        params[1].mul_(0.5)
    for _ in range(2):
        opt.step()
        for p in params:
            assert torch.equal(bf16_weight(p), p.detach().bfloat16())
    assert all(p._md_bf16_ver == p._version for p in params)
