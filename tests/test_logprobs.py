"""Token log probabilities, entropy, alternatives and their gradient against 64 bits.

Tolerances.  A thread adds at most 256 terms one after another and the joins add under 16 more, each
term carries a 2-ulp exp2 of an argument rounded three times: S is within (256 + 16 + 16) * 2^-24 =
1.8e-5 in the worst case, log S by the same amount absolutely; log p adds four fp32 roundings of its
own size, H four of log S.  A gradient is p (within twice that) times its bracket, rounded once to the
logits' type."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat

S_TOL = 1.8e-5
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 2.0**-149}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = float("inf")


def _reference(logits, tokens, temperature, top, ignore=-100):
    z = logits.detach().double()
    peak = z.max(-1).values
    empty = torch.isneginf(peak)
    z = (z - peak.masked_fill(empty, 0.0)[:, None]) / temperature  # (1e38 - 1e38 keeps no log of the count)
    logp = z - torch.logsumexp(z, -1).masked_fill(empty, 0.0)[:, None]
    p = logp.exp()
    scored = tokens != ignore
    lp = logp.gather(-1, tokens.masked_fill(~scored, 0)[:, None])[:, 0].masked_fill(~scored, 0.0)
    h = torch.special.entr(p).sum(-1)
    ids = logits.detach().double().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, h, logp.gather(-1, ids), ids, p, logp, scored, empty


def _near(got, ref, tol):
    got, ref = got.double(), ref.double()
    same = (got == ref) | (got.isnan() & ref.isnan())
    near = got.isfinite() & ref.isfinite() & ((got - ref).abs() <= tol)
    assert bool((same | near).all()), (got, ref)


def _check(logits, tokens, temperature=1.0, top=0, grads=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    m, dev = logits.shape[0], logits.device
    x = logits.detach().requires_grad_(grads)
    r = md.token_logprobs(x, tokens, temperature=temperature, top=top, entropy=True)
    lp, h, top_lp, ids, p, logp, scored, empty = _reference(logits, tokens, temperature, top)
    _near(r.logprobs, lp, S_TOL + 4 * 2.0**-24 * lp.abs())
    log_s = (logp.max(-1).values).abs()
    _near(r.entropy, h, S_TOL * (1 + 2 * h) + 4 * 2.0**-24 * log_s)
    if top:
        assert torch.equal(r.top_tokens, ids)
        _near(r.top_logprobs, top_lp, S_TOL + 4 * 2.0**-24 * top_lp.abs())
    if not grads:
        return r
    a, b, c = (torch.randn(*s, generator=g).to(dev) for s in ((m,), (m,), (m, max(top, 1))))
    outs, gs = [r.logprobs, r.entropy], [a, b]
    if top:
        outs, gs = outs + [r.top_logprobs], gs + [c]
    (d,) = torch.autograd.grad(outs, x, gs)
    named = torch.zeros_like(p)
    named.scatter_add_(-1, tokens.masked_fill(~scored, 0)[:, None], (a.double() * scored)[:, None])
    if top:
        named.scatter_add_(-1, ids, c.double())
    total = named.sum(-1, keepdim=True)
    plogp = -torch.special.entr(p)
    ref = (named - p * total - b.double()[:, None] * (plogp + p * h[:, None])) / temperature
    ref = ref.masked_fill(empty[:, None], 0.0)
    size = p * (total.abs() + named.abs().sum(-1, keepdim=True)) + b.double().abs()[:, None] * (-plogp + p * h[:, None])
    tol = HALF_ULP[d.dtype] * ref.abs() + (3 * S_TOL * size + 4 * 2.0**-24 * named.abs()) / temperature + TINY[d.dtype]
    assert d.dtype == logits.dtype and d.shape == logits.shape
    _near(d, ref, tol)
    if dev.type == "cuda":
        nat.check_status()
    return r


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (4, 20, 20), (2, 64, 64), (7, 503, 64),
                                            (33, 1001, 5), (150, 4099, 8), (2, 50257, 20), (300, 50257, 3),
                                            (1, 131072, 64), (1, 131071, 1)])
def test_values_and_gradients(device, dtype, rows, vocab, top):
    if device == "cpu" and rows * vocab > 3_000_000:
        pytest.skip("GPU size")
    g = torch.Generator().manual_seed(vocab)
    z = (torch.randn(rows, vocab, generator=g) * 3).to(device, dtype)
    t = torch.randint(0, vocab, (rows,), generator=g).to(device)
    t[::4] = -100 if rows > 4 else t[::4]
    _check(z, t, top=top)
    _check(z, t, top=min(top, 2), temperature=0.6)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start,pad", [(0, 7), (1, 0), (3, 2), (5, 11), (8, 8)])
def test_strides(device, dtype, start, pad):
    """Rows that start anywhere: the first and last logits of a row lie outside its 16-byte vectors."""
    rows, vocab = 6, 1237
    g = torch.Generator().manual_seed(5)
    buf = torch.randn(rows * (vocab + pad) + start, generator=g).to(device, dtype)
    z = buf[start:].as_strided((rows, vocab), (vocab + pad, 1), start)
    t = torch.tensor([0, 1, vocab - 1, vocab - 2, 7, 8], device=device)
    _check(z, t, top=9)
    wide = torch.randn(4, 5, 301, generator=g).to(device, dtype)
    _check(wide[:, -1], torch.tensor([0, 300, 4, 5], device=device), top=3)  # the last position of each sequence
    r = md.token_logprobs(wide, torch.zeros(4, 5, dtype=torch.long, device=device), top=2, entropy=True)
    flat = md.token_logprobs(wide.reshape(20, 301), torch.zeros(20, dtype=torch.long, device=device), top=2, entropy=True)
    assert r.top_tokens.shape == (4, 5, 2) and r.entropy.shape == (4, 5)
    assert all(torch.equal(x.reshape(y.shape), y) for x, y in zip(r, flat))
    col = torch.randn(301, 4, generator=g).to(device, dtype).t()  # vocabulary not contiguous
    _check(col, torch.tensor([0, 300, 4, 5], device=device), top=3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 777, 40000])
def test_masks(device, dtype, vocab):
    """-inf, the type's lowest value, rows with one or no logit left, equal logits, +inf and NaN."""
    g = torch.Generator().manual_seed(7)
    low = torch.finfo(dtype).min
    z = (torch.randn(9, vocab, generator=g) * 2).to(device, dtype)
    keep = (torch.rand(vocab, generator=g) < 0.5).to(device)
    z[0, ~keep] = -INF
    z[1, ~keep] = low
    z[2] = -INF  # nothing left
    z[3] = -INF
    z[3, vocab - 1] = 0.25  # one left
    z[4] = low
    z[5] = 1.5
    z[6] = -INF
    z[6, 0] = low
    z[7, 1] = torch.finfo(dtype).max
    t = torch.full((9,), vocab - 1, device=device)
    t[8] = -100
    top = min(vocab, 20)
    if dtype == torch.float32:
        z[7, 1] = 1e30
    _check(z, t, top=top)
    r = md.token_logprobs(z, t, top=top, entropy=True)
    assert r.logprobs[2] == -INF and r.entropy[2] == 0 and bool((r.top_logprobs[2] == -INF).all())
    assert r.logprobs[3] == 0 and r.entropy[3] == 0
    assert r.top_tokens[2].tolist() == r.top_tokens[5].tolist() == list(range(top))

    z[0, 2] = float("nan")
    z[1, 2] = INF
    z[7, 0] = INF
    z[7, 1] = INF
    x = z.clone().requires_grad_(True)
    r = md.token_logprobs(x, t, top=top, entropy=True)
    for row in (0, 1, 7):
        assert r.logprobs[row].isnan() and r.entropy[row].isnan() and bool(r.top_logprobs[row].isnan().all())
    assert r.top_tokens[1, 0] == 2 and r.top_tokens[7, :2].tolist() == [0, 1]
    assert bool(((r.top_tokens >= 0) & (r.top_tokens < vocab)).all())
    (d,) = torch.autograd.grad(r.logprobs, x, torch.ones_like(r.logprobs))
    assert bool(d[[0, 1, 7]].isnan().all()) and not bool(d[[2, 3, 4, 5, 6, 8]].isnan().any())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 200])
def test_alternatives_in_few_places(device, dtype, rows):
    """Orders that put the best logits next to each other, in steps of a thread's stride, or far more
    of them above the selection's first bound than it keeps at once."""
    if device == "cpu" and rows > 1:
        pytest.skip("GPU size")
    vocab = 50257
    i = torch.arange(vocab)
    crowd = torch.where((i // 32) % 128 < 19, 100.0 + (i % 977) * 0.5, (i % 61) * 0.125)  # whole lane groups
    for z in (i * 0.01, -i * 0.01, crowd, torch.where(i % 4096 < 8, 5.0 + i * 0.01, 0.0), torch.zeros(vocab)):
        z = z.to(device, dtype).expand(rows, vocab).contiguous()
        _check(z, torch.full((rows,), 11, device=device), top=20, grads=False)
        _check(z[:, 1:], torch.full((rows,), 11, device=device), top=64, grads=False)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    g = torch.Generator().manual_seed(11)
    z = torch.randn(6, 401, generator=g).to(device).requires_grad_(True)
    v = torch.randn(6, 401, generator=g).to(device)
    t = torch.tensor([0, 400, 17, -100, 5, 6], device=device)
    w = [torch.randn(s, generator=g).to(device) for s in ((6,), (6,), (6, 4))]

    def total(outs):
        return sum((o.double() * c.double()).sum() for o, c in zip(outs, w))

    r = md.token_logprobs(z, t, temperature=1.3, top=4, entropy=True)
    (d,) = torch.autograd.grad(total(r[:3]), z)

    def f(x):  # the alternatives as tokens: which four they are may change within the step
        y = md.token_logprobs(x, t, temperature=1.3, entropy=True)
        alt = [md.token_logprobs(x, r.top_tokens[:, i].contiguous(), temperature=1.3).logprobs for i in range(4)]
        return total([y.logprobs, y.entropy, torch.stack(alt, -1)])

    h = 5e-3
    with torch.no_grad():
        slope = (f(z + h * v) - f(z - h * v)) / (2 * h)
    # 36 outputs of size 10, each within 1e-6 of a smooth function: 36 * 1e-5 / h; third-order term
    # h^2 / 6 times a third derivative of size 36.
    assert abs(float(slope - (d.double() * v.double()).sum())) < 36 * 1e-6 / h + 36 * h * h


@pytest.mark.parametrize("device", DEVICES)
def test_partial_gradients_and_forms(device):
    z = torch.randn(4, 99, device=device).requires_grad_(True)
    t = torch.tensor([1, 2, 3, 4], device=device)
    r = md.token_logprobs(z, t)
    assert r.entropy is None and r.top_logprobs is None and r.top_tokens is None
    (d,) = torch.autograd.grad(r.logprobs.sum(), z)  # an expanded gradient
    ref = torch.nn.functional.one_hot(t, 99).double() - z.detach().double().softmax(-1)
    _near(d, ref, 2 * S_TOL + 2.0**-24)
    r = md.token_logprobs(z, t, entropy=True, top=3)
    (d,) = torch.autograd.grad(r.entropy.sum(), z, retain_graph=True)
    p = z.detach().double().softmax(-1)
    h = torch.special.entr(p).sum(-1, keepdim=True)
    _near(d, -p * (p.log() + h), 2 * S_TOL * h)
    (d,) = torch.autograd.grad(r.top_logprobs[:, 0].sum(), z)
    _near(d, torch.nn.functional.one_hot(z.argmax(-1), 99).double() - p, 2 * S_TOL + 2.0**-24)
    e = md.token_logprobs(z[:0], t[:0], entropy=True, top=2)
    assert e.logprobs.shape == (0,) and e.top_tokens.shape == (0, 2)
    assert torch.autograd.grad(e.logprobs.sum(), z)[0].abs().sum() == 0
    one = md.token_logprobs(z.detach()[0], t[0], top=1)  # a single row without a batch axis
    assert one.logprobs.shape == () and one.top_tokens.shape == (1,)


@pytest.mark.gpu
def test_token_outside_the_vocabulary_is_reported():
    nat.check_status()
    z = torch.randn(3, 50, device="cuda").requires_grad_(True)
    r = md.token_logprobs(z, torch.tensor([3, 50, -1], device="cuda"))
    assert not r.logprobs[0].isnan() and bool(r.logprobs[1:].isnan().all())
    torch.autograd.grad(r.logprobs.sum(), z)
    with pytest.raises(nat.NativeError, match="bad kernel argument"):
        nat.check_status()


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_other_stream():
    z = torch.randn(64, 50257, device="cuda").bfloat16()
    t = torch.randint(0, 50257, (64,), device="cuda")
    a = md.token_logprobs(z, t, top=20, entropy=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = md.token_logprobs(z * 1, t, top=20, entropy=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals():
    z, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.long)
    for bad in (
        lambda: md.token_logprobs(z.double(), t),
        lambda: md.token_logprobs(z, t[:2]),
        lambda: md.token_logprobs(z, t.int()),
        lambda: md.token_logprobs(z, t, temperature=0.0),
        lambda: md.token_logprobs(z, t, temperature=float("inf")),
        lambda: md.token_logprobs(z, t, top=11),
        lambda: md.token_logprobs(z, t, top=-1),
        lambda: md.token_logprobs(torch.zeros(3, 100), t, top=65),
        lambda: md.token_logprobs(z[:, :0], t),
        lambda: md.token_logprobs(z, t + 10),
    ):
        with pytest.raises((ValueError, TypeError, IndexError)):
            bad()
