"""Forward-mode derivatives of the operators: there, or refused; never lost."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import minidist as md

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_turns_tangents(device, grad, interleaved):
    """The operation is linear: a tangent turns as its primal does."""
    new = lambda h: torch.randn(2, 5, h, 16, device=device)  # noqa: E731
    q, k, dq, dk = new(4), new(2), new(4), new(2)
    table = md.rotary_table(12, 40, device=device)
    pos = torch.tensor([3, 0, 39, 7, 7], device=device)
    turn = lambda a, b: md.apply_rotary(a, b, table, pos, interleaved=interleaved)  # noqa: E731
    want_q, want_k = turn(dq, dk)
    if grad:
        q.requires_grad_(True)
    with forward_ad.dual_level():
        a, b = forward_ad.make_dual(q, dq), forward_ad.make_dual(k, dk)
        for x, y, tx, ty in ((a, b, want_q, want_k), (a, k, want_q, None), (q, b, None, want_k), (a, None, want_q, None)):
            for out, primal, want in zip(turn(x, y), turn(q, None if y is None else k), (tx, ty)):
                if out is None:
                    continue
                p, t = forward_ad.unpack_dual(out)
                assert torch.equal(p, primal)
                if want is None:
                    assert t is None or not t.any()
                else:
                    assert torch.equal(t, want)
        if not grad:
            with torch.no_grad():
                assert torch.equal(forward_ad.unpack_dual(turn(a, b)[0]).tangent, want_q)


@pytest.mark.parametrize("device", DEVICES)
def test_token_logprobs_refuse_tangents(device):
    z, t = torch.randn(3, 50, device=device), torch.tensor([1, 2, 3], device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(z, torch.randn_like(z))
        with pytest.raises(NotImplementedError, match="forward"):
            md.token_logprobs(dual, t, top=2, entropy=True)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            md.token_logprobs(dual[None], t[None])
        md.token_logprobs(z, t)
