"""Log probabilities of given tokens, with entropy and the best alternatives.

For each row of logits ``z`` and temperature ``T``::

    log p = z / T - logsumexp(z / T)        H = -sum_j p_j log p_j

:func:`token_logprobs` returns ``log p`` of one given token per row, and on request ``H`` and the
``top`` largest ``log p`` with their tokens (ties by the lower token).  All three differentiate::

    dz_j = (sum_i g_i ([j = t_i] - p_j) - g_H p_j (log p_j + H)) / T

On CUDA each direction is one sm_100a launch that reads the logits once (csrc/logprobs.cu); on CPU
the same arithmetic runs with torch operations.
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _native as nat

__all__ = ["TokenLogprobs", "token_logprobs"]

nat.declare("md_logprobs", "i:pp")
nat.declare("md_logprobs_backward", "i:pp")

MAX_TOP = 64
_COLDEST = 1e-37  # 1 / T and log2(e) / T have to be normal, finite fp32 numbers
_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # float32, the tokens' shape
    entropy: torch.Tensor | None  # float32, the tokens' shape
    top_logprobs: torch.Tensor | None  # float32 [..., top], largest first
    top_tokens: torch.Tensor | None  # int64 [..., top]


# struct MdLogprobsParams in csrc/logprobs.cu, field for field (native alignment): logits, ld, dtype,
# rows, vocab, tokens, ignore, inv_t, top, want_entropy, logprob, entropy, top_logprob, top_token,
# row_max, row_log, g_logprob, g_entropy, g_top, dlogits, ldd, status.
_PARAMS = struct.Struct("@Pq3iPqf2iPPPPPPPPPPqP")


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _call(entry, logits, tokens, temperature, top, ignore_index, logprob, h, top_lp, top_id, stats,
          g=None, gh=None, gt=None, out=None):
    row_max = _ptr(stats)
    params = _PARAMS.pack(logits.data_ptr(), logits.stride(0), _DTYPE_CODE[logits.dtype], *logits.shape,
                          tokens.data_ptr(), ignore_index, 1.0 / temperature, top, h is not None, _ptr(logprob),
                          _ptr(h), _ptr(top_lp), _ptr(top_id), row_max, row_max and row_max + 4 * logits.shape[0], _ptr(g), _ptr(gh),
                          _ptr(gt), _ptr(out), 0 if out is None else out.stride(0), nat.status_ptr(logits.device))
    with nat.on_device(logits):
        nat.check(getattr(nat.lib(), entry)(params, nat.stream_ptr()), entry)


def _forward(logits, tokens, temperature, top, entropy, ignore_index, for_backward):
    rows = logits.shape[0]
    new = logits.new_empty
    logprob = new(rows, dtype=torch.float32)
    h = new(rows, dtype=torch.float32) if entropy else None
    stats = new(2, rows, dtype=torch.float32) if for_backward else None  # per row: maximum, log of the sum
    top_lp = top_id = None
    if top:
        top_lp = torch.empty(rows, top, dtype=torch.float32, device=logits.device)
        top_id = torch.empty(rows, top, dtype=torch.int64, device=logits.device)
    if rows:
        _call("md_logprobs", logits, tokens, temperature, top, ignore_index, logprob, h, top_lp, top_id, stats)
    return logprob, h, top_lp, top_id, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top, entropy, ignore_index):
        ctx.set_materialize_grads(False)
        logprob, h, top_lp, top_id, stats = _forward(logits, tokens, temperature, top, entropy, ignore_index, True)
        ctx.save_for_backward(logits, tokens, h, top_id)
        ctx.how = (temperature, top, ignore_index, stats)
        if top_id is not None:
            ctx.mark_non_differentiable(top_id)
        return logprob, h, top_lp, top_id

    @staticmethod
    def backward(ctx, *grads):
        # (once_differentiable's wrapper only where a second derivative could be asked for)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, g, gh, gt, _):
    logits, tokens, h, top_id = ctx.saved_tensors
    temperature, top, ignore_index, stats = ctx.how
    rows, vocab = logits.shape
    # The kernel's vectors start equally far from a 16-byte boundary in logits and gradient: rows keep
    # the logits' padding modulo 16 bytes (the LM head's padded rows stay aligned) and the first one
    # its offset.
    size = logits.element_size()
    ld = vocab + (logits.stride(0) - vocab) % (16 // size)
    shift = logits.data_ptr() % 16 // size
    out = logits.new_empty(rows * ld + shift)[shift:].view(rows, ld) if shift else logits.new_empty(rows, ld)
    if ld != vocab:
        out = out[:, :vocab]
    if rows and (g is not None or gh is not None or gt is not None):
        g, gh, gt = (None if t is None else t.float().contiguous() for t in (g, gh, gt))
        _call("md_logprobs_backward", logits, tokens, temperature, top, ignore_index, None, h, None, top_id, stats,
              g, gh, gt, out)
    else:
        out.zero_()
    return out, None, None, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


class _Lookup(torch.autograd.Function):
    """The CPU form, with the same definitions at rows without a finite logit."""

    @staticmethod
    def forward(ctx, logits, tokens, temperature, top, entropy, ignore_index):
        ctx.set_materialize_grads(False)
        scored = tokens != ignore_index
        if bool((scored & ((tokens < 0) | (tokens >= logits.shape[1]))).any()):
            raise IndexError(f"token_logprobs: a token lies outside [0, {logits.shape[1]})")
        f = logits.float()
        peak = f.max(-1, keepdim=True).values
        empty = peak == float("-inf")
        z = (f - peak.masked_fill(empty, 0.0)) / temperature
        e = z.exp()
        total = e.sum(-1, keepdim=True)
        logp = (z - total.log()).masked_fill(empty, float("-inf"))
        p = (e / total).masked_fill(empty, 0.0)
        plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
        h = -plogp.sum(-1)
        at = tokens.masked_fill(~scored, 0)
        chosen = logp.gather(-1, at[:, None])[:, 0].masked_fill(~scored, 0.0)
        top_lp = top_id = None
        if top:
            order = f.masked_fill(f.isnan(), float("-inf")).sort(dim=-1, descending=True, stable=True)
            top_id = order.indices[:, :top].contiguous()
            top_lp = logp.gather(-1, top_id)
            ctx.mark_non_differentiable(top_id)
        ctx.saved = (p, plogp, h, scored, at, empty, top_id)
        ctx.how = (temperature, logits.dtype)
        return chosen, h if entropy else None, top_lp, top_id

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, gh, gt, _):
        p, plogp, h, scored, at, empty, top_id = ctx.saved
        temperature, dtype = ctx.how
        named = torch.zeros_like(p)
        if g is not None:
            named.scatter_add_(-1, at[:, None], g.masked_fill(~scored, 0.0)[:, None])
        if gt is not None:
            named.scatter_add_(-1, top_id, gt)
        d = named - p * named.sum(-1, keepdim=True)
        if gh is not None:
            d = d - gh[:, None] * (plogp + p * h[:, None])
        return (d.masked_fill(empty, 0.0) / temperature).to(dtype), None, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top: int = 0,
                   entropy: bool = False, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``tokens [...]`` under ``logits [..., vocab]`` at ``temperature``.

    Results are float32.  A row whose token is ``ignore_index`` gets 0 and passes no gradient from
    it (entropy and alternatives are computed for every row).  A row without any logit above
    ``-inf`` gives ``-inf``, entropy 0, the lowest tokens as alternatives and no gradient; a NaN or
    ``+inf`` logit makes its row's numbers NaN.  Logits may be a strided view with contiguous rows
    (the LM head's padded ones); one whose rows are not equally far apart, such as
    ``logits[:, :-1]`` of a batch, is copied (shift the tokens and ignore the last one instead).
    Of a tensor-parallel model gather the vocabulary first.  A token outside the vocabulary gives
    NaN, reported by :func:`minidist.ops._native.check_status` (on CPU it raises).  ``top`` is at
    most 64.  Differentiable once, in reverse mode.
    """
    if logits.dim() < 1 or logits.dtype not in _DTYPE_CODE:
        raise TypeError(f"token_logprobs: logits {tuple(logits.shape)} {logits.dtype} are not bfloat16, float16 or "
                        "float32 [..., vocab]")
    vocab = logits.shape[-1]
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1] or tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens {tuple(tokens.shape)} {tokens.dtype} are not int64 "
                         f"{tuple(logits.shape[:-1])} on {logits.device}")
    if vocab == 0:
        raise ValueError("token_logprobs: empty vocabulary")
    if not _COLDEST <= temperature <= 1.0 / _COLDEST:
        raise ValueError(f"token_logprobs: temperature {temperature} is not within [{_COLDEST}, {1.0 / _COLDEST:g}]")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: top={top} is not within [0, {min(MAX_TOP, vocab)}]")
    flat = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if flat.stride(1) != 1 or (flat.shape[0] > 1 and flat.stride(0) < vocab):
        flat = flat.contiguous()
    elif flat.shape[0] <= 1 and flat.stride(0) < vocab:
        flat = flat.as_strided(flat.shape, (vocab, 1))
    ids = tokens.contiguous() if tokens.dim() == 1 else tokens.reshape(-1).contiguous()
    # (A forward-mode tangent goes the same way, where torch says that there is no such derivative: a
    # kernel launch by itself would drop it.)
    need = (logits.requires_grad and torch.is_grad_enabled()) \
        or (nat.in_forward_mode() and forward_ad.unpack_dual(logits).tangent is not None)
    if not logits.is_cuda:
        out = _Lookup.apply(flat, ids, temperature, top, entropy, ignore_index)
    elif need:
        out = _TokenLogprobs.apply(flat, ids, temperature, top, entropy, ignore_index)
    else:
        out = _forward(flat, ids, temperature, top, entropy, ignore_index, False)[:4]
    lead = tokens.shape
    lp, h, top_lp, top_id = out
    if tokens.dim() != 1:
        lp = lp.view(lead)
        h = None if h is None else h.view(lead)
        top_lp = None if top_lp is None else top_lp.view(*lead, top)
        top_id = None if top_id is None else top_id.view(*lead, top)
    return TokenLogprobs(lp, h, top_lp, top_id)
