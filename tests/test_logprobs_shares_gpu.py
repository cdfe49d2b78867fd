"""Log probabilities without alternatives, at sizes where a row belongs to one, two or four warps or to a
cluster of blocks.

Tolerance.  A lane adds its logits in two sums; with one warp to a row that is vocab / 64 terms one after
another, each addition off by 2^-24 of the sum.  Beside them: the joins (under 16), a maximum that moves
(two roundings and an exp2 of 2 ulp each, ln of the row's length times: under 48), a term's own exp2 (4)
and its argument, four roundings of (z - m) / T, on average over p under ln(vocab) = 12 (48): together
under 128.  log S is off by as much absolutely, log p by four roundings of its own size more."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat

HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 2.0**-149}

#          1 row, a cluster of 8 ... 2; four warps; two; one
SIZES = [(1, 50257), (8, 50257), (33, 131072), (60, 50257), (100, 16411), (147, 9001), (300, 50257), (2000, 5003),
         (5000, 5003), (8192, 2500), (9472, 2051), (9500, 5003), (9500, 50257)]


def _near(got, ref, tol, what):
    off = (got.double() - ref).abs() - tol
    assert bool((off <= 0).all()), (what, float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_without_alternatives(rows, vocab, entropy, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    z = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    for at in range(0, rows, 1024):
        part = torch.randn(min(1024, rows - at), vocab, device="cuda", generator=g)
        z[at: at + 1024] = part * 3 + torch.linspace(-2, 2, vocab, device="cuda")  # the maximum moves on the way
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    z.requires_grad_(True)
    r = md.token_logprobs(z, t, entropy=entropy, temperature=0.9)
    assert (r.entropy is None) == (not entropy)
    a, b = (torch.randn(rows, device="cuda", generator=g) for _ in range(2))
    (d,) = torch.autograd.grad([r.logprobs, r.entropy] if entropy else [r.logprobs], z, [a, b] if entropy else [a])
    nat.check_status()
    s_tol = (vocab / 64 + 128) * 2.0**-24
    step = max(1, rows * vocab // 4_000_000)  # rows looked at
    for first in range(0, rows, 512 * step):
        i = torch.arange(first, min(rows, first + 512 * step), step, device="cuda")
        x = z.detach()[i].double() / 0.9
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        p, h = logp.exp(), torch.special.entr(logp.exp()).sum(-1)
        lp = logp.gather(-1, t[i, None])[:, 0]
        _near(r.logprobs[i], lp, s_tol + 4 * 2.0**-24 * lp.abs(), "log p")
        if entropy:
            _near(r.entropy[i], h, s_tol * (1 + 2 * h) + 4 * 2.0**-24 * logp.max(-1).values.abs(), "entropy")
        ga, gb = a[i, None].double(), b[i, None].double() * entropy
        named = torch.zeros_like(p).scatter_(-1, t[i, None], ga)
        plogp = -torch.special.entr(p)
        ref = (named - p * ga - gb * (plogp + p * h[:, None])) / 0.9
        size = (2 * p * ga.abs() + gb.abs() * (-plogp + p * h[:, None])) / 0.9
        _near(d[i], ref, HALF_ULP[dtype] * ref.abs() + 3 * s_tol * size + 4 * 2.0**-24 * named.abs() / 0.9 + TINY[dtype],
              "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 50, 300, 5000, 9500])
def test_the_split_of_a_row_changes_rounding_only(rows):
    """The same row by itself (a cluster's) and among others (one to four warps'); bit for bit the same in
    rows that start equally far from a 16-byte boundary (every eighth)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    z = (torch.randn(1, 8191, device="cuda", generator=g) * 4).bfloat16()
    t = torch.tensor([77], device="cuda")
    one = md.token_logprobs(z, t, entropy=True)
    many = md.token_logprobs(z.expand(rows, -1), t.expand(rows), entropy=True)
    tol = 2 * (8191 / 64 + 128) * 2.0**-24
    for x, y in zip(one[:2], many[:2]):
        assert float((x - y).abs().max()) < tol * (1 + 2 * float(x.abs()))
        assert torch.equal(y[8:], y[:-8])
    nat.check_status()
