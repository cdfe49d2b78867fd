"""Temperatures up to the ends of what fp32 can scale by."""

from __future__ import annotations

import pytest
import torch

import minidist as md

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_ends_of_the_range(device, grad):
    z = torch.tensor([[1.0, 3.0, -2.0, 3.0], [0.0, -1.0, 5.0, 2.0]], device=device).requires_grad_(grad)
    t = torch.tensor([1, 0], device=device)
    cold = md.token_logprobs(z, t, temperature=1e-37, entropy=True, top=2)  # the largest, shared where equal
    log2 = torch.tensor(2.0).log().item()
    assert abs(cold.logprobs[0].item() + log2) < 1e-6 and abs(cold.entropy[0].item() - log2) < 1e-6
    assert cold.logprobs[1].item() < -1e37 and cold.entropy[1].item() == 0.0
    hot = md.token_logprobs(z, t, temperature=1e37, entropy=True)  # all alike
    assert float((hot.logprobs + 2 * log2).abs().max()) < 1e-6 and float((hot.entropy - 2 * log2).abs().max()) < 1e-6
    if grad:
        (d,) = torch.autograd.grad(cold.logprobs[0], z)
        assert not d.isnan().any() and d[0, 1] > 1e36 and d[0, 3] < -1e36 and not d[0, ::2].any()


@pytest.mark.parametrize("bad", [0.0, -1.0, 1e-38, 4e-39, 1e-45, 5e-324, 1e38, 1e45, 1e300, float("inf"), float("nan")])
def test_beyond_it(bad):
    with pytest.raises(ValueError, match="temperature"):
        md.token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.long), temperature=bad)
