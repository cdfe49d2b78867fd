"""Tensors of more than 2^31 elements: offsets that 32 bits do not hold."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat

pytestmark = pytest.mark.gpu


def test_log_probabilities():
    rows, vocab = 43_000, 50_257
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    assert z.numel() > 2**31
    t = torch.arange(rows, device="cuda") % vocab
    g = torch.Generator(device="cuda").manual_seed(0)
    part = (torch.randn(1000, vocab, device="cuda", generator=g) * 3).bfloat16()
    with torch.no_grad():
        for at in range(0, rows, 1000):
            z[at: at + 1000] = part
    one = part.clone().requires_grad_(True)
    for top in (0, 5):
        r = md.token_logprobs(z, t, top=top, entropy=True)
        (d,) = torch.autograd.grad((r.logprobs.sum(), r.entropy.sum()), z)
        for at in (0, rows - 1000):  # the same logits by themselves
            q = md.token_logprobs(one, t[at: at + 1000], top=top, entropy=True)
            (e,) = torch.autograd.grad((q.logprobs.sum(), q.entropy.sum()), one)
            # sums over another number of warps: 1e-4 covers the longest chain (vocab / 64 * 2^-24) and its halving
            assert float((r.logprobs[at: at + 1000] - q.logprobs).abs().max()) < 1e-4
            assert float((r.entropy[at: at + 1000] - q.entropy).abs().max()) < 1e-4 * 25
            assert float((d[at: at + 1000].float() - e.float()).abs().max()) < 2.0**-8 + 1e-3
            if top:
                assert torch.equal(r.top_tokens[at: at + 1000], q.top_tokens)
        del d, r
    nat.check_status()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(interleaved):
    seq, heads, dim = 1 << 19, 52, 80
    q = torch.empty(1, seq, heads, dim, dtype=torch.bfloat16, device="cuda")
    assert q.numel() > 2**31
    part = torch.randn(1, 1024, heads, dim, device="cuda").bfloat16()
    for at in range(0, seq, 1024):
        q[:, at: at + 1024] = part
    table = md.rotary_table(40, seq, device="cuda")
    k = q[:, :, :1]
    y, z = md.apply_rotary(q, k, table, interleaved=interleaved)
    for at in (0, seq // 2, seq - 1024):
        want = md.apply_rotary(part, None, table, torch.arange(at, at + 1024, device="cuda"), interleaved=interleaved)[0]
        assert torch.equal(y[:, at: at + 1024], want) and torch.equal(z[:, at: at + 1024], want[:, :, :1])
    nat.check_status()
