"""Cases, inputs, plain forms and 64-bit definitions of the framework's language-model operators.

Operators: rotary positions (``minidist.apply_rotary``), log probabilities of given tokens with
entropy and top alternatives (``minidist.token_logprobs``), and the orthogonalised update of the
Muon optimizer (``minidist.orthogonalize``, ``minidist.ops.muon.muon_update_``).

``run`` with ``own = False`` computes them with elementary torch operations in 32 bits, rounded
once at the end; with ``own = True`` it makes the calls of the framework.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # quintic of the published Muon recipe
_EPS = 1e-7
_RMS = 0.2  # update RMS relative to lr, so that AdamW's learning rates carry over
IGNORE = -100


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def _rotary(name, batch, seq, heads, kv_heads, dim, rotary, dtype, *, interleaved=False, scaling="none",
            positions="start", packed=False, train=False):
    return {"op": "rotary", "name": name, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "dtype": dtype, "interleaved": interleaved, "scaling": scaling, "positions": positions,
            "packed": packed, "train": train}


def _logprobs(name, rows, vocab, dtype, *, top=0, entropy=True, temperature=1.0, masked=False, padded=False,
              train=False):
    return {"op": "logprobs", "name": name, "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "entropy": entropy, "temperature": temperature, "masked": masked, "padded": padded, "train": train}


def _muon(name, what, count, rows, cols, dtype):
    return {"op": "muon", "name": name, "what": what, "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # One training micro-batch of the 12-head, 768-wide GPT: q and k as they lie in the QKV
        # projection's output, forward and backward.
        _rotary("rotary train 16x1024 h12 d64", 16, 1024, 12, 12, 64, 64, "bf16", packed=True, train=True),
        # One new token for each of 32 sequences, shared key heads, half of each head rotated,
        # positions anywhere in a context stretched four times: launch latency.
        _rotary("rotary one token x32", 32, 1, 32, 8, 128, 64, "fp16", interleaved=True, scaling="linear",
                positions="scattered"),
        # A long prompt with the 80-wide heads of the 2.7B configuration, scaled by parts, ragged length.
        _rotary("rotary prompt 20011 h32 d80", 1, 20011, 32, 32, 80, 40, "bf16", scaling="yarn", positions="offset"),
        # Full precision, odd sizes, a rotary part that ends inside a vector.
        _rotary("rotary fp32 3x517 h5 d96", 3, 517, 5, 5, 96, 50, "fp32", interleaved=True, scaling="ntk",
                train=True),
        # Policy-gradient training step over the GPT-2 vocabulary: log probability and entropy of
        # the sampled tokens and the gradient of both, logits as the LM head stores them.
        _logprobs("logprobs train 8192x50257", 8192, 50257, "bf16", padded=True, train=True),
        # Scoring a batch of text with the 20 best alternatives of each position; rows of odd length.
        _logprobs("logprobs score 4096x50257 top20", 4096, 50257, "bf16", top=20),
        # The token just sampled, one sequence: latency.
        _logprobs("logprobs one token top5", 1, 50257, "fp32", top=5),
        # Constrained vocabulary, temperature, distillation from the top alternatives, one row
        # with nothing allowed.
        _logprobs("logprobs masked 333x32003 top8", 333, 32003, "fp16", top=8, temperature=0.7, masked=True,
                  train=True),
        # One square weight's update: latency of a chain of small products.
        _muon("orthogonalize 768x768", "orthogonalize", 1, 768, 768, "bf16"),
        # The QKV weights of all 12 layers of the 768-wide GPT, one optimizer step.
        _muon("muon step 12x 2304x768", "step", 12, 2304, 768, "fp32"),
        # A square weight of the 6.7B configuration.
        _muon("orthogonalize 4096x4096", "orthogonalize", 1, 4096, 4096, "bf16"),
        # Full precision in and out, ragged sizes.
        _muon("orthogonalize fp32 2x 203x1001", "orthogonalize", 2, 203, 1001, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotary", "logprobs", "muon"))
    if op == "rotary":
        one = rng.random() < 0.3
        dim = rng.choice((32, 64, 80, 96, 128))
        heads = rng.choice((1, 2, 5, 12, 16, 20, 25, 32))
        kv = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        batch = _log_int(rng, 1, 256) if one else rng.randint(1, 8)
        seq = 1 if one else _log_int(rng, 2, min(32768, 12_000_000 // (batch * heads * dim)))
        packed = kv == heads and rng.random() < 0.5
        return {k: v for k, v in _rotary(
            "", batch, seq, heads, kv, dim, dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2),
            rng.choice(("bf16", "fp16", "fp32")), interleaved=rng.random() < 0.5,
            scaling=rng.choice(("none", "linear", "ntk", "yarn")),
            positions="scattered" if one else rng.choice(("start", "offset", "scattered")),
            packed=packed, train=not one and rng.random() < 0.5).items() if k != "name"}
    if op == "logprobs":
        vocab = _log_int(rng, 500, 131072)
        return {k: v for k, v in _logprobs(
            "", _log_int(rng, 1, min(8192, 200_000_000 // vocab)), vocab, rng.choice(("bf16", "fp16", "fp32")),
            top=rng.choice((0, 0, 1, 5, 20, 32)), entropy=rng.random() < 0.7,
            temperature=rng.choice((1.0, 1.0, 0.7, 1.3)), masked=rng.random() < 0.3, padded=rng.random() < 0.5,
            train=rng.random() < 0.5).items() if k != "name"}
    what = rng.choice(("orthogonalize", "orthogonalize", "step"))
    dtype = "fp32" if what == "step" else rng.choice(("bf16", "fp16", "fp32"))
    small = _log_int(rng, 48, 1600)
    # (A full-precision answer is only asked of wide matrices: a square one's smallest singular
    # values amplify fp32's own rounding past fp32.)
    large = _log_int(rng, 2 * small if what == "orthogonalize" and dtype == "fp32" else small, 6400)
    rows, cols = (small, large) if rng.random() < 0.5 else (large, small)
    count = rng.randint(1, max(1, min(12, 8_000_000_000 // (small * small * large))))
    return {k: v for k, v in _muon("", what, count, rows, cols, dtype).items() if k != "name"}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _max_positions(case):
    return {"start": case["seq"], "offset": case["seq"] + 1500, "scattered": 32768}[case["positions"]]


def _angles(case):
    """(angle of each pair per unit of position, factor on cos and sin), 64 bits."""
    r, base, factor, original = case["rotary"], 10000.0, 4.0, 8192
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk" and r > 2:
        base = base * factor ** (r / (r - 2))
    inv = base ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return inv / factor, 1.0
    if case["scaling"] == "yarn":
        lo = r * math.log(original / (32 * 2 * math.pi)) / (2 * math.log(base))
        hi = r * math.log(original / (1 * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv / factor * (1 - keep) + inv * keep, 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _prepare_rotary(case, g):
    b, s, h, hk, d = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    dt = _DTYPES[case["dtype"]]
    n = _max_positions(case)
    inv, factor = _angles(case)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    table = (torch.stack([angle.cos(), angle.sin()], -1) * factor).float()
    if case["packed"]:  # q and k where the QKV projection leaves them: [.., head, (q, k, v), dim]
        qkv = torch.randn(b, s, h, 3, d, device="cuda", generator=g).to(dt)
        q, k = qkv[:, :, :, 0], qkv[:, :, :, 1]
    else:
        q = torch.randn(b, s, h, d, device="cuda", generator=g).to(dt)
        k = torch.randn(b, s, hk, d, device="cuda", generator=g).to(dt)
    if case["positions"] == "start":
        positions = None
    elif case["positions"] == "offset":
        positions = torch.arange(1500, 1500 + s, device="cuda")
    else:
        positions = torch.randint(0, n, (b, s), device="cuda", generator=g)
    state = {"q": q, "k": k, "table": table, "positions": positions}
    if case["train"]:
        state["q"], state["k"] = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        state["dq"] = torch.randn(b, s, h, d, device="cuda", generator=g).to(dt)
        state["dk"] = torch.randn(b, s, hk, d, device="cuda", generator=g).to(dt)
    return state


def _prepare_logprobs(case, g):
    m, v = case["rows"], case["vocab"]
    dt = _DTYPES[case["dtype"]]
    ld = (v + 7) // 8 * 8 if case["padded"] else v
    buf = torch.empty(m, ld, dtype=dt, device="cuda")
    logits = buf[:, :v]
    # Rows of different sharpness, from nearly flat to nearly decided.
    sharp = torch.exp(0.4 * torch.randn(m, 1, device="cuda", generator=g)) * 2.5
    at = 0
    while at < m:  # in pieces, so that the 32-bit draw stays small
        z = torch.randn(min(1024, m - at), v, device="cuda", generator=g)
        logits[at: at + 1024] = (z * sharp[at: at + 1024]).to(dt)
        at += 1024
    tokens = torch.randint(0, v, (m,), device="cuda", generator=g)
    if case["masked"]:  # columns that a grammar forbids, and one row where it allows nothing
        allowed = torch.rand(v, device="cuda", generator=g) < 0.7
        logits.masked_fill_(~allowed, float("-inf"))
        if m > 2:
            logits[m // 2] = float("-inf")
    if m > 4:  # prompt positions, not scored
        tokens[:: 5] = IGNORE
    state = {"logits": logits, "tokens": tokens}
    if case["train"]:
        state["logits"] = logits.detach().requires_grad_(True)
        state["g"] = torch.randn(m, device="cuda", generator=g) / m
        state["ge"] = torch.randn(m, device="cuda", generator=g) * (0.01 / m)
        state["gt"] = torch.randn(m, max(1, case["top"]), device="cuda", generator=g) * (0.1 / m)
    return state


def _gradient(rows, cols, g):
    """A weight gradient as backward makes it: output gradients times inputs over tokens that share
    directions, features of different scale."""
    t = 2 * min(rows, cols)
    z = torch.randn(t, 32, device="cuda", generator=g)
    x = torch.randn(t, cols, device="cuda", generator=g) + 0.5 * z @ torch.randn(32, cols, device="cuda", generator=g)
    dy = torch.randn(t, rows, device="cuda", generator=g) + 0.3 * z @ torch.randn(32, rows, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))
    dy *= torch.exp(0.5 * torch.randn(rows, device="cuda", generator=g))
    return dy.t() @ x * (1e-4 / t)


def _prepare_muon(case, g):
    c, m, n = case["count"], case["rows"], case["cols"]
    if case["what"] == "orthogonalize":
        if case["dtype"] == "fp32":
            u = torch.randn(c, m, n, device="cuda", generator=g)
        else:
            u = torch.stack([_gradient(m, n, g) for _ in range(c)])
            u = u / u.std()
        return {"u": u.to(_DTYPES[case["dtype"]])}
    return {"params": [0.1 * torch.randn(m, n, device="cuda", generator=g) for _ in range(c)],
            "grads": [_gradient(m, n, g) for _ in range(c)],
            "momenta": [8.0 * _gradient(m, n, g) for _ in range(c)]}


def prepare(case, seed):
    g = _gen(seed)
    state = {"rotary": _prepare_rotary, "logprobs": _prepare_logprobs, "muon": _prepare_muon}[case["op"]](case, g)
    state["case"] = dict(case)
    return state


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    f = x.float()
    if interleaved:
        a, b = f[..., 0:r:2], f[..., 1:r:2]
    else:
        a, b = f[..., : r // 2], f[..., r // 2: r]
    p, q = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([y, f[..., r:]], -1).to(x.dtype)


@torch.no_grad()
def _plain_rotary(case, s):
    positions = s["positions"]
    cs = s["table"][: case["seq"]] if positions is None else s["table"][positions]
    cos, sin = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    il = case["interleaved"]
    out = [_turn(s["q"], cos, sin, il), _turn(s["k"], cos, sin, il)]
    if case["train"]:  # the gradient of a rotation is the rotation back
        out += [_turn(s["dq"], cos, -sin, il), _turn(s["dk"], cos, -sin, il)]
    return out


@torch.no_grad()
def _plain_logprobs(case, s):
    logits, tokens, top = s["logits"], s["tokens"], case["top"]
    m, v = logits.shape
    z = logits.float() / case["temperature"]
    peak = z.max(-1, keepdim=True).values
    empty = peak == float("-inf")
    z = z - torch.where(empty, torch.zeros_like(peak), peak)
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    logp = z - total.log()
    logp = torch.where(empty, torch.full_like(logp, float("-inf")), logp)
    p = torch.where(empty, torch.zeros_like(e), e / total)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    h = -plogp.sum(-1)
    counted = tokens != IGNORE
    at = torch.where(counted, tokens, torch.zeros_like(tokens))
    chosen = logp.gather(-1, at[:, None])[:, 0]
    out = {"logprobs": torch.where(counted, chosen, torch.zeros_like(chosen))}
    if case["entropy"]:
        out["entropy"] = h
    if top:
        # Largest first, ties by the lowest index: one key of value and index (32-bit floats
        # order like their bits once the negative ones are flipped).
        bits = (logits.float() + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 32) | (v - 1 - torch.arange(v, device=logits.device))
        best = v - 1 - (key.topk(top, -1).values & 0xFFFFFFFF)
        out["top_logprobs"], out["top_tokens"] = logp.gather(-1, best), best
    if case["train"]:
        # z_j / T: d logp_t = [j = t] - p_j, d H = -p_j (logp_j + H)
        g = torch.where(counted, s["g"], torch.zeros_like(s["g"]))
        both = g + s["gt"].sum(-1) if top else g
        d = -p * both[:, None]
        if case["entropy"]:
            d = d - s["ge"][:, None] * (plogp + p * h[:, None])
        d.scatter_add_(-1, at[:, None], g[:, None])
        if top:
            d.scatter_add_(-1, best, s["gt"])
        d = torch.where(empty, torch.zeros_like(d), d / case["temperature"])
        out["dlogits"] = d.to(logits.dtype)
    return out


def _plain_orthogonal(u):
    a, b, c = _COEFFICIENTS
    x = u.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + _EPS)
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _hyper(case):
    return {"lr": 3e-4, "momentum": 0.95, "weight_decay": 0.1}


@torch.no_grad()
def _plain_muon(case, s):
    if case["what"] == "orthogonalize":
        return _plain_orthogonal(s["u"]).to(s["u"].dtype)
    hp = _hyper(case)
    lr, mu, wd = hp["lr"], hp["momentum"], hp["weight_decay"]
    torch._foreach_mul_(s["momenta"], mu)
    torch._foreach_add_(s["momenta"], s["grads"])
    u = torch.stack(torch._foreach_add(s["grads"], s["momenta"], alpha=mu))
    o = _plain_orthogonal(u)
    torch._foreach_mul_(s["params"], 1 - lr * wd)
    torch._foreach_add_(s["params"], list(o.unbind()), alpha=-lr * _RMS * math.sqrt(max(case["rows"], case["cols"])))
    return {"params": s["params"], "momenta": s["momenta"]}


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------


def _own_rotary(case, s):
    import minidist as md

    q, k = md.apply_rotary(s["q"], s["k"], s["table"], s["positions"], interleaved=case["interleaved"])
    if not case["train"]:
        return [q, k]
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return [q.detach(), k.detach(), dq, dk]


def _own_logprobs(case, s):
    import minidist as md

    r = md.token_logprobs(s["logits"], s["tokens"], temperature=case["temperature"], top=case["top"],
                          entropy=case["entropy"], ignore_index=IGNORE)
    out = {"logprobs": r.logprobs.detach()}
    outs, grads = [r.logprobs], [s.get("g")]
    if case["entropy"]:
        out["entropy"] = r.entropy.detach()
        outs, grads = outs + [r.entropy], grads + [s.get("ge")]
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs.detach(), r.top_tokens
        outs, grads = outs + [r.top_logprobs], grads + [s.get("gt")]
    if case["train"]:
        (out["dlogits"],) = torch.autograd.grad(outs, s["logits"], grads)
    return out


def _own_muon(case, s):
    import minidist as md
    from minidist.ops.muon import muon_update_

    if case["what"] == "orthogonalize":
        return md.orthogonalize(s["u"])
    muon_update_(s["params"], s["grads"], s["momenta"], **_hyper(case))
    return {"params": s["params"], "momenta": s["momenta"]}


def run(state):
    case = state["case"]
    plain = {"rotary": _plain_rotary, "logprobs": _plain_logprobs, "muon": _plain_muon}
    kernels = {"rotary": _own_rotary, "logprobs": _own_logprobs, "muon": _own_muon}
    return (kernels if own else plain)[case["op"]](case, state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    if case["op"] == "rotary":
        size = _DTYPES[case["dtype"]].itemsize
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"])
        ways = 2 if case["train"] else 1
        rows = case["seq"] if case["positions"] != "scattered" else min(tokens, _max_positions(case))
        other = rows * case["rotary"] * 4 + (0 if case["positions"] == "start" else 8 * tokens)
        return {"bytes": ways * 2 * n * case["dim"] * size + other, "flops": ways * n * case["rotary"] * 3}
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        size = _DTYPES[case["dtype"]].itemsize
        small = case["rows"] * (8 + 4 + 4 * case["entropy"] + 12 * case["top"])
        if case["train"]:
            small += case["rows"] * (4 + 4 * case["entropy"] + 4 * case["top"])
        return {"bytes": n * size * (2 if case["train"] else 1) + small, "flops": n * (9 if case["train"] else 5)}
    small, large = sorted((case["rows"], case["cols"]))
    c = case["count"]
    n = c * small * large
    # Symmetric products need one triangle.
    flops = 5 * c * (small * (small + 1) * large + small * small * (small + 1) + 2 * small * small * large)
    return {"bytes": n * (2 * _DTYPES[case["dtype"]].itemsize if case["what"] == "orthogonalize" else 20), "flops": flops}


# ---------------------------------------------------------------------------
# Definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_rotary(case, s):
    inv, factor = _angles(case)
    positions = s["positions"]
    if positions is None:
        positions = torch.arange(case["seq"], device="cuda")
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"),
                       positions.double()[..., None, None] * inv)  # [.., seq, 1, pairs]
    r = case["rotary"]

    def spin(x, by):
        y = x.detach().double().clone()
        part = y[..., :r].reshape(*y.shape[:-1], *((r // 2, 2) if case["interleaved"] else (2, r // 2)))
        pairs = part if case["interleaved"] else part.mT
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        y[..., :r] = (z if case["interleaved"] else z.mT).reshape(*y.shape[:-1], r)
        return y

    out = [spin(s["q"], turn), spin(s["k"], turn)]
    if case["train"]:
        out += [spin(s["dq"], turn.conj()), spin(s["dk"], turn.conj())]
    return out


def _exact_logprobs(case, s):
    top, pieces = case["top"], []
    for at in range(0, case["rows"], 512):
        part = slice(at, at + 512)
        raw = s["logits"].detach()[part]
        z = raw.double() / case["temperature"]
        lse = torch.logsumexp(z, -1)
        empty = torch.isneginf(lse)
        logp = (z - lse.masked_fill(empty, 0.0)[:, None])
        p = logp.exp()
        h = torch.special.entr(p).sum(-1)
        tokens = s["tokens"][part]
        scored = tokens != IGNORE
        rows = torch.arange(len(tokens), device="cuda")
        got = {"logprobs": logp[rows, tokens.clamp(min=0)].masked_fill(~scored, 0.0)}
        if case["entropy"]:
            got["entropy"] = h
        if top:
            order = raw.double().sort(dim=-1, descending=True, stable=True).indices[:, :top]
            got["top_logprobs"], got["top_tokens"] = logp.gather(-1, order), order
        if case["train"]:
            want = torch.zeros_like(z)  # the gradient with respect to each log probability
            want[rows[scored], tokens[scored]] = s["g"][part][scored].double()
            if top:
                want.scatter_add_(-1, order, s["gt"][part].double())
            d = want - p * want.sum(-1, keepdim=True)
            if case["entropy"]:
                d += s["ge"][part].double()[:, None] * (torch.special.entr(p) - p * h[:, None])
            got["dlogits"] = d.masked_fill(empty[:, None], 0.0) / case["temperature"]
        pieces.append(got)
    return {k: torch.cat([x[k] for x in pieces]) for k in pieces[0]}


def _exact_orthogonal(u):
    """Through the Gram matrix of the shorter side: the same polynomial of the singular values."""
    a, b, c = _COEFFICIENTS
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + _EPS)
    left = x.shape[-2] <= x.shape[-1]
    for _ in range(5):
        w = x @ x.mT if left else x.mT @ x
        w = torch.baddbmm(a * torch.eye(w.shape[-1], dtype=w.dtype, device=w.device).expand_as(w),
                          w, b * torch.eye(w.shape[-1], dtype=w.dtype, device=w.device) + c * w)
        x = w @ x if left else x @ w
    return x


def _exact_muon(case, s):
    if case["what"] == "orthogonalize":
        return _exact_orthogonal(s["u"])
    hp = _hyper(case)
    params, momenta = [], []
    for w, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = hp["momentum"] * m.double() + g.double()
        o = _exact_orthogonal((g.double() + hp["momentum"] * m)[None])[0]
        params.append(w.double() - hp["lr"] * (hp["weight_decay"] * w.double() + _RMS * math.sqrt(max(w.shape)) * o))
        momenta.append(m)
    return {"params": params, "momenta": momenta}


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "logprobs": _exact_logprobs, "muon": _exact_muon}[case["op"]](case, state)
