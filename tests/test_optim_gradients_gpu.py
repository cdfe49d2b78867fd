"""Gradients that do not lie as their parameters do, in FusedAdamW's kernels."""

from __future__ import annotations

import pytest
import torch

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
