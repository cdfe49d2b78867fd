"""Orthogonalised updates: Newton-Schulz products and the Muon step around them.

``X = U / (|U|_F + eps)``, then ``steps`` times (for the shorter side's Gram matrix)::

    A = X X^T        X = a X + (b A + c A A) X

drives every singular value of ``U`` towards one and leaves its singular vectors
(Jordan et al. 2024).  :func:`orthogonalize` is that alone; :func:`muon_update_` adds momentum and
the weights' update, for many matrices at once; :class:`minidist.optim.Muon` is the optimizer.

On CUDA equally shaped matrices go through one chain of launches on the tensor cores
(csrc/muon.cu): the momentum pass, the norm, three products a step, the last of which updates the
weights in its epilogue.  On CPU the same arithmetic runs with torch operations.
"""

from __future__ import annotations

import ctypes
import functools
import math
from collections.abc import Sequence

import torch

from . import _native as nat

__all__ = ["orthogonalize", "muon_update_", "COEFFICIENTS"]

nat.declare("md_muon", "i:pp")
nat.declare("md_muon_workspace", "l:iiii")

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_BATCH = 64
_WORKSPACE = 4 << 30  # bytes at most, unless one matrix takes more
_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class _Params(ctypes.Structure):
    """Mirror of ``struct MdMuonParams`` in csrc/muon.cu."""

    _fields_ = [
        ("count", ctypes.c_int),
        ("rows", ctypes.c_int),
        ("cols", ctypes.c_int),
        ("dtype", ctypes.c_int),
        ("step", ctypes.c_int),
        ("split", ctypes.c_int),
        ("iterations", ctypes.c_int),
        ("a", ctypes.c_float),
        ("b", ctypes.c_float),
        ("c", ctypes.c_float),
        ("eps", ctypes.c_float),
        ("momentum", ctypes.c_float),
        ("nesterov", ctypes.c_int),
        ("decay", ctypes.c_float),
        ("rate", ctypes.c_float),
        ("lr", ctypes.c_void_p),
        ("inv_scale", ctypes.c_void_p),
        ("skip", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_longlong),
        ("tile", ctypes.c_int),
        ("status", ctypes.c_void_p),
        ("src", ctypes.c_void_p * _BATCH),
        ("m", ctypes.c_void_p * _BATCH),
        ("out", ctypes.c_void_p * _BATCH),
        ("shadow", ctypes.c_void_p * _BATCH),
    ]


def _params(count, rows, cols, dtype, split, steps, coefficients, eps, device):
    p = _Params()
    p.count, p.rows, p.cols, p.dtype, p.split, p.iterations = count, rows, cols, dtype, split, steps
    p.a, p.b, p.c = coefficients
    p.eps = eps
    size = nat.lib().md_muon_workspace(count, rows, cols, split)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = workspace.data_ptr(), size
    p.status = nat.status_ptr(device)
    return p, workspace


def _per_call(rows: int, cols: int, split) -> int:
    """Matrices updated together: batches are for small ones, whose tiles do not fill the SMs one by one,
    and their workspace (both parts of X twice, A and B) must not grow with a large model (six of
    16384 x 4096 take 22 to 25 ms whether by 1, by 3 or together, and 0.6, 1.7 or 3.4 GiB)."""
    return max(1, min(_BATCH, _WORKSPACE // max(1, nat.lib().md_muon_workspace(1, rows, cols, split))))


def _check_polynomial(steps, coefficients, eps) -> None:
    if steps < 1 or len(coefficients) != 3 or not eps >= 0.0:
        raise ValueError(f"Newton-Schulz: steps={steps}, coefficients={coefficients}, eps={eps}: expected at least one "
                         "step, three coefficients and a non-negative eps")


@functools.lru_cache(maxsize=64)
def _stays_in_range(steps: int, a: float, b: float, c: float) -> bool:
    """Whether X, A = X X^T and B = b A + c A A fit the products' fp16 operands (2^12 times their
    value, below 65504) at every step, for any matrix: singular values start within one, the
    polynomial's largest value bounds the next step's."""
    top = 1.0
    for _ in range(steps):
        values = [top * i / 1024 for i in range(1025)]
        grams = [s * s for s in values]
        seconds = [b * g + c * g * g for g in grams]
        if not all(abs(v) < 15.5 for v in (top, grams[-1], *seconds)):  # (of 15.99: what rounding may add)
            return False
        top = max(abs(s * (a + f)) for s, f in zip(values, seconds))
    return True


def _check_range(steps, coefficients) -> None:
    if not _stays_in_range(steps, *map(float, coefficients)):
        raise ValueError(f"Newton-Schulz: coefficients={tuple(coefficients)} take singular values below one out of the "
                         f"range of the products' operands within {steps} steps")


def _orthogonal_cpu(u: torch.Tensor, steps, coefficients, eps) -> torch.Tensor:
    a, b, c = coefficients
    x = u.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _orthogonalize_cuda(u: torch.Tensor, steps, coefficients, eps, tile: int = 0, precise: bool = False) -> torch.Tensor:
    rows, cols = u.shape[-2:]
    u = u.contiguous()
    out = torch.empty_like(u)
    count = u.numel() // (rows * cols)
    # A bf16 answer is rounded more coarsely than one product of fp16 parts errs; fp16 and fp32
    # answers take the three-product form.
    split = precise or u.dtype != torch.bfloat16
    size = rows * cols * u.element_size()
    together = _per_call(rows, cols, split)
    for at in range(0, count, together):
        n = min(together, count - at)
        p, workspace = _params(n, rows, cols, _DTYPE_CODE[u.dtype], split, steps, coefficients, eps, u.device)
        p.tile = tile
        src, dst = u.data_ptr() + at * size, out.data_ptr() + at * size
        p.src[:n] = [src + i * size for i in range(n)]
        p.out[:n] = [dst + i * size for i in range(n)]
        with nat.on_device(u):
            nat.check(nat.lib().md_muon(ctypes.addressof(p), nat.stream_ptr()), "md_muon")
        del workspace  # (reused only by later work of this stream)
    return out


def orthogonalize(u: torch.Tensor, *, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                  eps: float = 1e-7, precise: bool = False) -> torch.Tensor:
    """``u [..., rows, cols]`` (bfloat16, float16 or float32) with its singular values driven towards
    one, each matrix by itself, in ``u``'s type.

    The polynomial ``a s + b s^3 + c s^5`` has to keep ``|s| <= 1.3`` within about two, as the default
    and the classical ``(1.5, -0.5, 0)`` and ``(15/8, -10/8, 3/8)`` do; one that could leave the range of
    the kernels' operands (``s^2`` or ``b s^2 + c s^4`` of 15.5) is refused on CUDA.  bfloat16 results
    are within a bfloat16 rounding or so of exact, float16 and float32 ones within their own type's;
    ``precise`` takes those types' products (three of fp16 parts each instead of one) for bfloat16 as
    well, whose results are then off by their rounding alone.  Not differentiable."""
    if u.dim() < 2 or u.dtype not in _DTYPE_CODE:
        raise TypeError(f"orthogonalize: {tuple(u.shape)} {u.dtype} is not a bfloat16, float16 or float32 matrix")
    _check_polynomial(steps, coefficients, eps)
    u = u.detach()
    if u.numel() == 0:
        return u.clone()
    if not u.is_cuda:
        return _orthogonal_cpu(u, steps, coefficients, eps).to(u.dtype)
    _check_range(steps, coefficients)
    return _orthogonalize_cuda(u, steps, coefficients, eps, precise=precise)


def _check_step(params, grads, momenta, shadows) -> None:
    if not len(params) == len(grads) == len(momenta) or (shadows is not None and len(shadows) != len(params)):
        raise ValueError("muon_update_: params, grads, momenta (and shadows) differ in number")
    for i, (w, g, m) in enumerate(zip(params, grads, momenta)):
        if w.dim() != 2 or w.dtype != torch.float32 or not w.is_contiguous():
            raise ValueError(f"muon_update_: parameter {i} {tuple(w.shape)} {w.dtype} is not a contiguous float32 matrix")
        if g.shape != w.shape or g.dtype != torch.float32 or g.device != w.device:
            raise ValueError(f"muon_update_: gradient {i} {tuple(g.shape)} {g.dtype} does not go with {tuple(w.shape)}")
        if m.shape != w.shape or m.dtype != torch.float32 or m.device != w.device or not m.is_contiguous():
            raise ValueError(f"muon_update_: momentum {i} is not a contiguous float32 {tuple(w.shape)}")
        sh = None if shadows is None else shadows[i]
        if sh is not None and (sh.shape != w.shape or sh.dtype != torch.bfloat16 or sh.device != w.device
                               or not sh.is_contiguous()):
            raise ValueError(f"muon_update_: shadow {i} is not a contiguous bfloat16 {tuple(w.shape)}")


def _check_scalar(t, name: str, device) -> None:
    """The kernels read one float through the pointer: nothing else may stand there."""
    if isinstance(t, torch.Tensor) and (t.numel() != 1 or t.dtype != torch.float32 or t.device != device):
        raise ValueError(f"muon_update_: {name} {tuple(t.shape)} {t.dtype} on {t.device} is not one float32 on {device}")


def _scale(rows: int, cols: int, rms: float) -> float:
    # An orthogonal [rows, cols] has entries of size 1 / sqrt(max(rows, cols)).
    return rms * math.sqrt(max(rows, cols))


def _step_cuda(params, grads, momenta, shadows, lr, momentum, nesterov, weight_decay, steps, coefficients, eps, rms,
               inv_scale, skip, precise, tile: int = 0) -> None:
    """Up to ``_BATCH`` equally shaped matrices of one device, checked by the caller."""
    n, device = len(params), params[0].device
    rows, cols = params[0].shape
    # One product of fp16 parts, unless asked otherwise: X errs by 1e-3 or 2e-3 of itself, and the weights
    # take lr rms of it.
    p, workspace = _params(n, rows, cols, _DTYPE_CODE[torch.float32], precise, steps, coefficients, eps, device)
    p.tile, p.step, p.momentum, p.nesterov = tile, 1, momentum, nesterov
    factor = _scale(rows, cols, rms)
    if isinstance(lr, torch.Tensor):
        p.lr, p.decay, p.rate = lr.data_ptr(), weight_decay, factor
    else:
        p.decay, p.rate = 1.0 - lr * weight_decay, lr * factor
    p.inv_scale, p.skip = nat.ptr(inv_scale), nat.ptr(skip)
    held = [g.contiguous() for g in grads]
    p.src[:n] = [g.data_ptr() for g in held]
    p.m[:n] = [m.data_ptr() for m in momenta]
    p.out[:n] = [w.data_ptr() for w in params]
    if shadows is not None:
        p.shadow[:n] = [nat.ptr(sh) for sh in shadows]
    with nat.on_device(params[0]):
        nat.check(nat.lib().md_muon(ctypes.addressof(p), nat.stream_ptr()), "md_muon")
    del workspace, held  # (reused only by later work of this stream)
    # The kernels write through raw pointers: say so, as an in-place operation of torch's does, to
    # autograd (saved tensors) and to whoever keeps copies by version (the fused block's bf16 weights).
    torch.autograd.graph.increment_version([*params, *momenta])
    if shadows is not None:
        torch.autograd.graph.increment_version([sh for sh in shadows if sh is not None])


@torch.no_grad()
def muon_update_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], *,
                 lr: float | torch.Tensor, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7, rms: float = 0.2,
                 shadows: Sequence[torch.Tensor | None] | None = None, inv_scale: torch.Tensor | None = None,
                 skip: torch.Tensor | None = None, precise: bool = False) -> None:
    """One Muon step on fp32 matrices, in place::

        m = momentum m + g        u = g + momentum m  (m without nesterov)
        w = (1 - lr weight_decay) w - lr rms sqrt(max(rows, cols)) orthogonalize(u)

    so that an update's entries have size ``lr rms`` whatever the shape (0.2 is AdamW's usual size,
    whose learning rates then carry over).  ``lr`` may be a float32 tensor of one element on the
    device.  ``shadows``: bfloat16 copies to refresh with the weights.  ``inv_scale`` / ``skip``: the
    loss scaler's device factor on the gradients and its flag that leaves everything unchanged, each
    one float32 on the parameters' device.  Everything is checked before anything changes.  The
    versions of what is written go up, as with torch's own in-place operations.
    Matrices of one shape and device are updated together, up to 64 and 4 GiB of workspace at a time.

    On CUDA an update comes from single products of fp16 parts and is off by about 2e-3 of itself;
    ``precise`` takes three products, as for a float32 :func:`orthogonalize`: off by 1e-5 or less, in 2.1
    to 2.7 times the time (12 x 2304 x 768 469 and 1061 us, 1600 x 6400 396 and 1077)."""
    _check_polynomial(steps, coefficients, eps)
    _check_step(params, grads, momenta, shadows)
    groups: dict = {}
    for i, w in enumerate(params):
        groups.setdefault((w.shape, w.device), []).append(i)
    for device in {device for _, device in groups}:
        for name, t in (("lr", lr), ("inv_scale", inv_scale), ("skip", skip)):
            _check_scalar(t, name, device)
        if device.type == "cuda":
            _check_range(steps, coefficients)
    for (shape, device), members in groups.items():
        rows, cols = shape
        if rows * cols == 0:
            continue
        if device.type != "cuda":
            if skip is not None and bool(skip.item()):
                continue
            for i in members:
                g = grads[i] if inv_scale is None else grads[i] * inv_scale
                momenta[i].mul_(momentum).add_(g)
                u = g.add(momenta[i], alpha=momentum) if nesterov else momenta[i]
                x = _orthogonal_cpu(u, steps, coefficients, eps)
                params[i].mul_(1 - lr * weight_decay).sub_(x * (lr * _scale(rows, cols, rms)))
                if shadows is not None and shadows[i] is not None:
                    shadows[i].copy_(params[i])
            continue
        together = _per_call(rows, cols, precise)
        for at in range(0, len(members), together):
            part = members[at: at + together]
            _step_cuda(*([t[i] for i in part] for t in (params, grads, momenta)),
                       None if shadows is None else [shadows[i] for i in part], lr, momentum, nesterov, weight_decay,
                       steps, coefficients, eps, rms, inv_scale, skip, precise)
