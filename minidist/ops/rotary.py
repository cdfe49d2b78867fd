"""Rotary positions: cos / sin tables and their application to query and key heads.

A pair ``(a, b)`` of channels of a token at position ``p`` turns by ``p * f_i``::

    a' = a cos(p f_i) - b sin(p f_i)        f_i = base ** (-2 i / rotary_dim)
    b' = b cos(p f_i) + a sin(p f_i)

The first ``rotary_dim`` channels of each head turn, the others pass through.  On CUDA
:func:`apply_rotary` is one sm_100a launch for queries and keys together
(csrc/rotary.cu), on CPU the same arithmetic with torch operations; both
differentiate (the gradient is the rotation back) in either mode.
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _native as nat

__all__ = ["RotaryScaling", "rotary_table", "apply_rotary"]

nat.declare("md_rotary", "i:pp")

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@dataclass(frozen=True)
class RotaryScaling:
    """How frequencies are stretched for contexts ``factor`` times longer than trained.

    ``kind``: ``"linear"`` divides every position by ``factor`` (position interpolation);
    ``"ntk"`` raises the base to ``base * factor ** (r / (r - 2))``; ``"yarn"`` interpolates
    per frequency, keeping those that turn more than ``beta_fast`` times over
    ``original_positions``, dividing those that turn less than ``beta_slow`` times and blending
    in between, and multiplies cos and sin by ``0.1 ln(factor) + 1``.
    """

    kind: str = "linear"
    factor: float = 1.0
    original_positions: int = 8192
    beta_fast: float = 32.0
    beta_slow: float = 1.0

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"RotaryScaling kind {self.kind!r}: expected 'linear', 'ntk' or 'yarn'")
        if not 1.0 <= self.factor < math.inf:
            raise ValueError(f"RotaryScaling factor {self.factor}: expected a finite value of at least 1")
        if self.original_positions < 1 or not 0.0 < self.beta_slow <= self.beta_fast < math.inf:
            raise ValueError(f"RotaryScaling original_positions={self.original_positions}, beta_fast={self.beta_fast}, "
                             f"beta_slow={self.beta_slow}: expected at least one position and 0 < beta_slow <= beta_fast")


def rotary_table(rotary_dim: int, positions: int, *, base: float = 10000.0, scaling: RotaryScaling | None = None,
                 device=None) -> torch.Tensor:
    """``[positions, rotary_dim / 2, 2]`` fp32 (cos, sin), computed in 64 bits and rounded once."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim={rotary_dim}: expected a positive even number")
    if positions < 0 or not base > 0:
        raise ValueError(f"positions={positions}, base={base}: expected non-negative and positive")
    r, scale = rotary_dim, 1.0
    pair = torch.arange(r // 2, dtype=torch.float64, device=device)
    if scaling is not None and scaling.kind == "ntk" and r > 2:
        base = base * scaling.factor ** (r / (r - 2))
    freq = base ** (-2.0 * pair / r)
    if scaling is not None and scaling.kind == "linear":
        freq = freq / scaling.factor
    elif scaling is not None and scaling.kind == "yarn":
        def pair_turning(times: float) -> float:  # the pair that turns so often over the original context
            return r * math.log(scaling.original_positions / (2 * math.pi * times)) / (2 * math.log(base))

        lo = max(math.floor(pair_turning(scaling.beta_fast)), 0)
        hi = min(math.ceil(pair_turning(scaling.beta_slow)), r - 1)
        stretch = ((pair - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - stretch) + freq / scaling.factor * stretch
        scale = 0.1 * math.log(scaling.factor) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], dim=-1) * scale).float()


# struct MdRotaryParams in csrc/rotary.cu, field for field (native alignment): x[2], y[2], xs[2][3],
# ys[2][3], heads[2], table, table_rows, positions, positions64, ps[2], batch, seq, dim, rotary,
# interleaved, inverse, dtype, status.
_PARAMS = struct.Struct("@2P2P6q6q2iPqPi2q7iP")


def _launch(q, k, q_out, k_out, table, positions, interleaved: bool, inverse: bool) -> None:
    B, S, H, D = q.shape
    xs, ys = q.stride()[:3], q_out.stride()[:3]
    if k is None:
        kp, kop, Hk, kxs, kys = 0, 0, 0, (0, 0, 0), (0, 0, 0)
    else:
        kp, kop, Hk, kxs, kys = k.data_ptr(), k_out.data_ptr(), k.shape[2], k.stride()[:3], k_out.stride()[:3]
    if positions is None:
        pos, wide, ps = 0, 0, (0, 0)
    else:
        pos, wide, ps = positions.data_ptr(), positions.dtype == torch.int64, positions.stride()
        if len(ps) == 1:
            ps = (0, ps[0])
    half = table.shape[1]
    if table.data_ptr() % (8 if half % 2 else 16):  # (a slice of rows starts where the kernel can)
        table = table.clone()
    params = _PARAMS.pack(q.data_ptr(), kp, q_out.data_ptr(), kop, *xs, *kxs, *ys, *kys, H, Hk, table.data_ptr(),
                          table.shape[0], pos, wide, *ps, B, S, D, 2 * half, interleaved, inverse,
                          _DTYPE_CODE[q.dtype], nat.status_ptr(q.device))
    with nat.on_device(q):
        nat.check(nat.lib().md_rotary(params, nat.stream_ptr()), "md_rotary")


def _turn_cpu(x, table, positions, interleaved, inverse):
    if positions is None:
        cs = table[: x.shape[1]]
    else:
        positions = positions.long()
        if x.device.type == "cpu" and bool(((positions < 0) | (positions >= table.shape[0])).any()):
            raise IndexError(f"apply_rotary: a position lies outside [0, {table.shape[0]})")
        cs = table[positions]
    cos, sin = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    if inverse:
        sin = -sin
    r = 2 * table.shape[1]
    f = x.float()
    a, b = (f[..., 0:r:2], f[..., 1:r:2]) if interleaved else (f[..., : r // 2], f[..., r // 2: r])
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, f[..., r:]], -1).to(x.dtype)


def _turn(q, k, table, positions, interleaved, inverse, inplace=False):
    if not q.is_cuda:
        out = [None if t is None else _turn_cpu(t, table, positions, interleaved, inverse) for t in (q, k)]
        if not inplace:
            return out
        for t, o in zip((q, k), out):
            if t is not None:
                t.copy_(o)
        return [q, k]
    if inplace:
        q_out, k_out = q, k
    else:
        if q.stride(-1) != 1:
            q = q.contiguous()
        q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), None
        if k is not None:
            if k.stride(-1) != 1:
                k = k.contiguous()
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    _launch(q, k, q_out, k_out, table, positions, interleaved, inverse)
    return [q_out, k_out]


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, table, positions, interleaved, inverse):
        ctx.save_for_backward(table, positions)
        ctx.how = (interleaved, inverse)
        if nat.in_forward_mode():
            ctx.save_for_forward(table, positions)
            ctx.shapes = (q.shape, None if k is None else k.shape)
        ctx.set_materialize_grads(False)
        return tuple(_turn(q, k, table, positions, interleaved, inverse))

    @staticmethod
    def backward(ctx, dq, dk):
        table, positions = ctx.saved_tensors
        interleaved, inverse = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() else _turn  # (differentiable again if asked for)
        if dq is not None:
            dq, dk = turn(dq, dk, table, positions, interleaved, not inverse)
        elif dk is not None:
            dk, _ = turn(dk, None, table, positions, interleaved, not inverse)
        return dq, dk, None, None, None, None


    @staticmethod
    def jvp(ctx, q, k, *_):  # tangents: the operation is linear
        table, positions = ctx.saved_tensors
        if q is None:
            return k.new_zeros(ctx.shapes[0]), _turn(k, None, table, positions, *ctx.how)[0]
        turned, other = _turn(q, k, table, positions, *ctx.how)
        return turned, q.new_zeros(ctx.shapes[1]) if k is None and ctx.shapes[1] is not None else other


def _has_tangent(t: torch.Tensor | None) -> bool:
    """Whether ``t`` carries a forward-mode tangent, which a kernel launch by itself would drop."""
    return t is not None and forward_ad.unpack_dual(t).tangent is not None


def _check(q, k, table, positions) -> None:
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("apply_rotary expects q and k of [batch, seq, heads, head_dim]")
    if q.dtype not in _DTYPE_CODE:
        raise TypeError(f"apply_rotary: dtype {q.dtype} is not bfloat16, float16 or float32")
    if k is not None and (k.dtype != q.dtype or k.device != q.device or k.shape[:2] != q.shape[:2]
                          or k.shape[3] != q.shape[3]):
        raise ValueError(f"apply_rotary: k {tuple(k.shape)} {k.dtype} does not go with q {tuple(q.shape)} {q.dtype}")
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous() \
            or table.device != q.device or not 0 < 2 * table.shape[1] <= q.shape[3]:
        raise ValueError(f"apply_rotary: table {tuple(table.shape)} {table.dtype} is not a contiguous float32 "
                         f"[positions, rotary_dim / 2, 2] on {q.device} with rotary_dim <= {q.shape[3]}")
    if table.requires_grad and torch.is_grad_enabled():
        raise ValueError("apply_rotary: the table requires a gradient, but gets none (it is a constant here)")
    if positions is None:
        if q.shape[1] > table.shape[0]:
            raise ValueError(f"apply_rotary: {q.shape[1]} tokens, but the table has {table.shape[0]} positions")
    elif positions.dtype not in (torch.int64, torch.int32) or positions.device != q.device \
            or tuple(positions.shape) not in ((q.shape[1],), tuple(q.shape[:2])):
        raise ValueError(f"apply_rotary: positions {tuple(positions.shape)} {positions.dtype} are not int32 / int64 "
                         f"[seq] or [batch, seq] on {q.device}")


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, table: torch.Tensor, positions: torch.Tensor | None = None,
                 *, interleaved: bool = False):
    """Queries ``[B, S, H, D]`` and keys ``[B, S, Hk, D]`` (or None) at their positions.

    ``table``: from :func:`rotary_table`; its width says how many channels turn.  ``positions``:
    int32 / int64 ``[S]`` or ``[B, S]``, by default 0, 1, .. S - 1.  ``interleaved`` pairs
    neighbouring channels, otherwise a channel pairs with the one ``rotary_dim / 2`` further.
    The inputs may be strided views (a packed QKV projection); the results are contiguous.  A
    position outside the table makes its token's turned channels NaN and is reported by
    :func:`minidist.ops._native.check_status` (on CPU it raises).
    """
    _check(q, k, table, positions)
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) \
            or (nat.in_forward_mode() and (_has_tangent(q) or _has_tangent(k))):
        return _Rotary.apply(q, k, table, positions, interleaved, False)
    return tuple(_turn(q, k, table, positions, interleaved, False))


def rotate_packed_(qkv: torch.Tensor, heads: int, table: torch.Tensor, *, batch: int, inverse: bool = False):
    """Turn the queries and keys of a packed ``[batch * seq, heads * (q, k, v) * dim]`` projection in
    place (``inverse``: turn a packed gradient back).  No autograd: the fused block calls it in both
    directions."""
    rows, cols = qkv.shape
    seq, dim = rows // batch, cols // (3 * heads)
    view = qkv.as_strided((batch, seq, heads, 3, dim),
                          (seq * qkv.stride(0), qkv.stride(0), 3 * dim, dim, 1), qkv.storage_offset())
    q, k = view[:, :, :, 0], view[:, :, :, 1]
    _check(q, k, table, None)
    _turn(q, k, table, None, False, inverse, inplace=True)
    if qkv.is_cuda:  # written through a raw pointer
        torch.autograd.graph.increment_version(qkv)
    return qkv
