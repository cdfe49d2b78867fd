"""Optimizers.

:class:`FusedAdamW` is ``torch.optim.AdamW`` (same hyper-parameters, same
update, same ``state_dict`` keys ``step``/``exp_avg``/``exp_avg_sq``) executed
as one multi-tensor sm_100a kernel per parameter group (csrc/optim.cu).  The
kernel also refreshes the bf16 shadow weights the fused GEMMs read, so the
next forward does not pay for a separate cast.  Off CUDA it runs the same
arithmetic with torch ops, so CPU tests exercise identical semantics.

``capturable=True`` keeps each group's learning rate and step count in device
memory ([lr, t]; the kernel computes the bias corrections), so a training step
captured in a CUDA graph (:class:`minidist.graphs.GraphedStep`) advances the
step on every replay; :meth:`FusedAdamW.sync_hyperparams` refreshes the device
learning rate from ``param_groups`` between replays.

:class:`Muon` is FusedAdamW with orthogonalised momentum updates
(:mod:`minidist.ops.muon`) for the parameter groups that hold matrices;
:func:`muon_groups` sorts a model's parameters into the two kinds of group.
"""

from __future__ import annotations

import math
import warnings

import torch

from .ddp import wait_handle
from .ops import _native as nat
from .ops import grads as gradsink
from .ops import muon as muon_ops

__all__ = ["FusedAdamW", "Muon", "muon_groups"]


class FusedAdamW(torch.optim.Optimizer):
    # Parameters whose DDP all-reduce is still in flight (``_md_grad_event``) are
    # updated last, after waiting on exactly their handle (DistributedDataParallel's
    # ``defer_last_buckets``); the global step guard in minidist.ddp leaves them to us.
    honours_grad_events = True

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, capturable: bool = False):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("invalid AdamW hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._tables: dict[int, tuple] = {}
        self.capturable = capturable
        self._hp: dict[int, torch.Tensor] = {}  # capturable: device [lr, step] per group
        self._hp_lr: dict[int, float] = {}

    def sync_hyperparams(self) -> None:
        """Copy each group's current ``lr`` into its device slot (capturable mode; call between
        graph replays -- it launches work, so not while a graph is being captured)."""
        for gi, hp in self._hp.items():
            lr = float(self.param_groups[gi]["lr"])
            if self._hp_lr.get(gi) != lr:
                hp[0:1].fill_(lr)
                self._hp_lr[gi] = lr

    def state_dict(self):
        # In capturable mode the step count advances on the device; bring it to the host state.
        for gi, hp in self._hp.items():
            t = float(hp[1].item())
            for p in self.param_groups[gi]["params"]:
                st = self.state.get(p)
                if st and "step" in st:
                    st["step"].fill_(t)
        return super().state_dict()

    # -- state ----------------------------------------------------------------------

    def _state(self, p: torch.Tensor) -> dict:
        st = self.state[p]
        if not st:
            st["step"] = torch.zeros((), dtype=torch.float32)
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        return st

    def _init_states(self, params) -> None:
        """First step of CUDA fp32 parameters: their moments as views of two flat zeroed buffers
        (two fills for the whole group instead of two per parameter; 16-byte-aligned slices)."""
        todo = [p for p in params if not self.state[p] and p.is_cuda and p.dtype == torch.float32]
        if not todo:
            return
        sizes = [(p.numel() + 3) // 4 * 4 for p in todo]
        flat = torch.zeros(2, sum(sizes), dtype=torch.float32, device=todo[0].device)
        off = 0
        for p, n in zip(todo, sizes):
            st = self.state[p]
            st["step"] = torch.zeros((), dtype=torch.float32)
            st["exp_avg"] = flat[0, off: off + p.numel()].view_as(p)
            st["exp_avg_sq"] = flat[1, off: off + p.numel()].view_as(p)
            off += n

    # -- step -----------------------------------------------------------------------

    @torch.no_grad()
    def check_nonfinite(self, flag: torch.Tensor) -> None:
        """Set device ``flag`` (float32 ``[1]``) to 1 if any gradient is inf / NaN, without a host
        synchronisation (one read-only multi-tensor pass per parameter group; CPU parameters are
        checked with torch ops)."""
        for gi, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if group.get("orthogonal"):
                self._wait_for(params)
            fused = [p for p in params if p.is_cuda and p.dtype == torch.float32 and p.grad.dtype == torch.float32]
            fused_ids = {id(p) for p in fused}
            for p in params:
                if id(p) not in fused_ids:
                    flag.add_((~torch.isfinite(p.grad)).any().to(flag.dtype).to(flag.device))
            if group.get("orthogonal"):
                if fused:
                    table, chunk_t, n = self._table(("grads", gi), fused, moments=False)
                    nat.check(nat.lib().md_nonfinite(table.data_ptr(), chunk_t.data_ptr(), n, flag.data_ptr(),
                                                     nat.stream_ptr()), "md_nonfinite")
                continue
            self._init_states(fused)  # the kernel table points at the moments too
            if fused:
                for key, part in self._partitions(gi, fused):
                    table, chunk_t, n = self._table(key, part)
                    nat.check(nat.lib().md_nonfinite(table.data_ptr(), chunk_t.data_ptr(), n, flag.data_ptr(),
                                                     nat.stream_ptr()), "md_nonfinite")

    def _partitions(self, gi, fused):
        late = [p for p in fused if getattr(p, "_md_grad_event", None) is not None]
        if not late:
            return [(gi, fused)]
        early = [p for p in fused if getattr(p, "_md_grad_event", None) is None]
        return [((gi, 0), early), ((gi, 1), late)] if early else [((gi, 1), late)]

    @torch.no_grad()
    def step(self, closure=None, *, inv_scale: torch.Tensor | None = None, skip: torch.Tensor | None = None):
        """One AdamW step.  ``inv_scale`` / ``skip`` (device float32 ``[1]``, from
        :class:`minidist.amp.DistributedGradScaler`): gradients are multiplied by ``inv_scale``
        inside the update kernel, and the whole update is skipped on the device when ``skip``
        is nonzero -- the loss scaler's unscale and overflow skip with no extra pass over the
        gradients and no host synchronisation."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_scaler(inv_scale, skip)
        self._scaler_ptrs = (None if inv_scale is None else inv_scale.data_ptr(),
                             None if skip is None else skip.data_ptr())
        for gi, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if group.get("orthogonal"):
                self._orthogonal_step(gi, group, params, inv_scale, skip)
                continue
            self._init_states(params)
            states = [self._state(p) for p in params]
            # One multi-tensor op for every parameter's step count (a per-tensor
            # loop of CPU adds cost ~0.6 ms of host time per step at GPT-2 size).
            torch._foreach_add_([st["step"] for st in states], 1.0)
            t = float(states[0]["step"])
            b1, b2 = group["betas"]
            lr, eps, wd = group["lr"], group["eps"], group["weight_decay"]
            bc1 = 1.0 - b1**t
            bc2_sqrt = math.sqrt(1.0 - b2**t)
            cuda = [p.is_cuda and p.dtype == torch.float32 and p.grad.dtype == torch.float32 for p in params]
            fused = [p for p, c in zip(params, cuda) if c]
            rest = [p for p, c in zip(params, cuda) if not c]
            hp = None
            if self.capturable and fused:
                hp = self._hp.get(gi)
                if hp is None:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("FusedAdamW(capturable=True) needs one eager step before capture")
                    hp = torch.tensor([lr, t - 1.0], dtype=torch.float32, device=fused[0].device)
                    self._hp[gi], self._hp_lr[gi] = hp, float(lr)
                if not torch.cuda.is_current_stream_capturing():
                    self.sync_hyperparams()
                hp[1:2].add_(1.0)
            if rest and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdamW: only CUDA fp32 parameters can be stepped inside a CUDA graph")
            if fused:
                # Parameters whose gradient all-reduce is still in flight (DDP with
                # defer_last_buckets) are updated last, after waiting on its event.
                late = [p for p in fused if getattr(p, "_md_grad_event", None) is not None]
                if late:
                    early = [p for p in fused if getattr(p, "_md_grad_event", None) is None]
                    if early:
                        self._fused_update((gi, 0), early, lr, b1, b2, eps, wd, bc1, bc2_sqrt, hp)
                    for ev in {id(p._md_grad_event): p._md_grad_event for p in late}.values():
                        wait_handle(ev)
                    for p in late:
                        p._md_grad_event = None
                    self._fused_update((gi, 1), late, lr, b1, b2, eps, wd, bc1, bc2_sqrt, hp)
                else:
                    self._fused_update(gi, fused, lr, b1, b2, eps, wd, bc1, bc2_sqrt, hp)
                self._ensure_grad_buffers()
            for ev in {id(h): h for h in (getattr(p, "_md_grad_event", None) for p in rest) if h is not None}.values():
                wait_handle(ev)
            if rest and skip is not None and bool(skip.item()):
                rest = []
            for p in rest:
                p._md_grad_event = None
                st = self.state[p]
                g = p.grad.to(p.dtype)
                if inv_scale is not None:
                    g = g * inv_scale.to(g.device)
                p.mul_(1 - lr * wd)
                st["exp_avg"].mul_(b1).add_(g, alpha=1 - b1)
                st["exp_avg_sq"].mul_(b2).addcmul_(g, g, value=1 - b2)
                denom = st["exp_avg_sq"].sqrt().div_(bc2_sqrt).add_(eps)
                p.addcdiv_(st["exp_avg"], denom, value=-lr / bc1)
        return loss

    def _check_scaler(self, *scalars: torch.Tensor | None) -> None:
        """The update kernels read one float through each pointer: refused, before any group is
        updated, unless that is what it points at."""
        scalars = [t for t in scalars if t is not None]
        if not scalars:
            return
        devices = {p.device for g in self.param_groups for p in g["params"] if p.is_cuda and p.grad is not None}
        for t in scalars:
            if t.numel() != 1 or (devices and (t.dtype != torch.float32 or devices != {t.device})):
                raise ValueError(f"inv_scale / skip {tuple(t.shape)} {t.dtype} on {t.device} is not one float32 on the "
                                 f"parameters' device ({', '.join(map(str, devices)) or 'cpu'})")

    @staticmethod
    def _wait_for(params) -> None:
        """Order the current stream after the gradient reductions of ``params`` that are in flight."""
        late = [p for p in params if getattr(p, "_md_grad_event", None) is not None]
        for ev in {id(p._md_grad_event): p._md_grad_event for p in late}.values():
            wait_handle(ev)
        for p in late:
            p._md_grad_event = None

    def _ensure_grad_buffers(self) -> None:
        """Give every CUDA fp32 parameter without one a persistent gradient buffer.

        Fused kernels write gradients into these views (ops/grads.py), so the
        gradient pointers stay fixed from step to step and the device-side
        parameter table is built once.  Parameters that a wrapper (DDP) has
        already given a buffer keep it.
        """
        if getattr(self, "_grad_buffers_done", False):
            return
        self._grad_buffers_done = True
        todo = [p for g in self.param_groups for p in g["params"]
                if p.is_cuda and p.dtype == torch.float32 and gradsink.main_grad(p) is None]
        if not todo:
            return
        align = 64
        sizes = [(p.numel() + align - 1) // align * align for p in todo]
        flat = torch.zeros(sum(sizes), dtype=torch.float32, device=todo[0].device)
        off = 0
        for p, n in zip(todo, sizes):
            view = flat[off: off + p.numel()].view_as(p)
            if p.grad is not None:
                view.copy_(p.grad)
                p.grad = view
            gradsink.set_main_grad(p, view)
            off += n
        self._grad_flat = flat

    def _fused_update(self, gi, params, lr, b1, b2, eps, wd, bc1, bc2_sqrt, hp=None) -> None:
        table, chunk_t, n = self._table(gi, params)
        inv_ptr, skip_ptr = getattr(self, "_scaler_ptrs", (None, None))
        rc = nat.lib().md_adamw(table.data_ptr(), chunk_t.data_ptr(), n, lr, b1, b2, eps, wd, bc1, bc2_sqrt,
                                inv_ptr, skip_ptr, 0, nat.stream_ptr(), None if hp is None else hp.data_ptr())
        nat.check(rc, "md_adamw")
        # (The kernel leaves the versions as they are, so the bf16 copies that it refreshed stay valid, and
        # those that it was not given because they were stale stay stale.)

    def _table(self, gi, params, moments: bool = True):
        """Device (tensor, chunk) table of ``params`` for the multi-tensor kernels, cached per key
        while the pointers stay the same (``moments=False``: for passes over the gradients alone)."""
        from .models.fused_gpt import _SHADOW, _SHADOW_VER

        lib = nat.lib()
        rows, key = [], []
        for p in params:
            st = self.state[p] if moments else None
            if not p.grad.is_contiguous():  # (kept: the kernel reads it through the table)
                p.grad = p.grad.contiguous()
            g = p.grad
            sh = getattr(p, _SHADOW, None)
            if sh is not None and (sh.shape != p.shape or getattr(p, _SHADOW_VER, None) != p._version):
                sh = None  # stale shadow: let the next forward recast it
            m, v = (st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()) if moments else (0, 0)
            ptrs = (p.data_ptr(), g.data_ptr(), m, v, sh.data_ptr() if sh is not None else 0, p.numel())
            rows.append(ptrs)
            key.append(ptrs)
        key = tuple(key)
        cached = self._tables.get(gi)
        dev = params[0].device
        if cached is None or cached[0] != key:
            chunk = lib.md_adamw_chunk()
            chunks = [(i, c) for i, p in enumerate(params) for c in range(-(-p.numel() // chunk))]
            # Pinned sources: a copy from pageable memory is not allowed inside a graph capture.
            table_h = torch.tensor(rows, dtype=torch.int64).pin_memory()
            chunk_h = torch.tensor(chunks, dtype=torch.int32).pin_memory()
            table = table_h.to(dev, non_blocking=True)
            chunk_t = chunk_h.to(dev, non_blocking=True)
            cached = (key, table, chunk_t, len(chunks), table_h, chunk_h)
            self._tables[gi] = cached
        return cached[1], cached[2], cached[3]


class Muon(FusedAdamW):
    """Muon (Jordan et al. 2024) for matrices, AdamW for everything else, in one optimizer.

    A group with ``orthogonal=True`` holds 2-D fp32 parameters; each takes
    ``w = (1 - lr weight_decay) w - lr rms sqrt(max(rows, cols)) X`` where ``X`` is the
    orthogonalised momentum (:func:`minidist.ops.muon.muon_update_`).  ``rms`` is the size of an
    update's entries per unit of ``lr``; 0.2, about AdamW's, lets both kinds of group share a
    learning rate.  ``precise`` takes products of fp32's precision on CUDA.  Other groups are
    FusedAdamW's.  A group that does not say is orthogonal if all its parameters are matrices (a warning
    tells of matrices that a mixed one leaves to AdamW)::

        opt = Muon(muon_groups(model), lr=3e-4)

    State: ``momentum_buffer`` per matrix, AdamW's elsewhere.  Under tensor parallelism a shard is
    orthogonalised as a matrix of its own.  FSDP's flat shards hold pieces of matrices: they are
    refused, unless a group says ``orthogonal=False``.  The loss scaler, deferred DDP buckets and
    ``capturable=True`` work as with FusedAdamW.
    """

    def __init__(self, params, lr: float = 3e-4, *, momentum: float = 0.95, nesterov: bool = True, rms: float = 0.2,
                 ns_steps: int = 5, ns_coefficients=muon_ops.COEFFICIENTS, betas=(0.9, 0.95), eps: float = 1e-8,
                 weight_decay: float = 1e-2, capturable: bool = False, precise: bool = False):
        if not 0 <= momentum < 1 or not rms > 0 or ns_steps < 1 or len(ns_coefficients) != 3:
            raise ValueError("invalid Muon hyper-parameters")
        # add_param_group (called by the base constructor) completes each group from these
        self._matrix_defaults = dict(momentum=momentum, nesterov=nesterov, rms=rms, ns_steps=ns_steps,
                                     ns_coefficients=tuple(ns_coefficients), precise=precise)
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable)

    def add_param_group(self, group: dict) -> None:
        params = group["params"]
        group["params"] = params = [params] if isinstance(params, torch.Tensor) else list(params)
        params = [p[1] if isinstance(p, tuple) else p for p in params]  # (named parameters)
        matrices = [p.dim() == 2 and p.dtype == torch.float32 for p in params]
        if "orthogonal" not in group:
            _refuse_flat_shards(params)
            group["orthogonal"] = all(matrices)
            if any(matrices) and not all(matrices):
                warnings.warn(f"Muon: a group of {len(params)} parameters holds {sum(matrices)} matrices and others, so all "
                              "of it takes AdamW; sort them with muon_groups(model) or say orthogonal=False", stacklevel=3)
        if group["orthogonal"]:
            if not all(matrices):
                bad = next(p for p, ok in zip(params, matrices) if not ok)
                raise ValueError(f"Muon: a {tuple(bad.shape)} {bad.dtype} parameter is not a float32 matrix; put it in a "
                                 "group with orthogonal=False")
            for k, v in self._matrix_defaults.items():
                group.setdefault(k, v)
        super().add_param_group(group)

    def _orthogonal_step(self, gi, group, params, inv_scale, skip) -> None:
        from .models.fused_gpt import _SHADOW, _SHADOW_VER

        self._wait_for(params)
        lr = group["lr"]
        cuda = params[0].is_cuda
        if self.capturable and cuda:
            capturing = torch.cuda.is_current_stream_capturing()
            if gi not in self._hp:
                if capturing:
                    raise RuntimeError("Muon(capturable=True) needs one eager step before capture")
                self._hp[gi] = torch.tensor([lr, 0.0], dtype=torch.float32, device=params[0].device)
                self._hp_lr[gi] = float(lr)
            if not capturing:
                self.sync_hyperparams()
            lr = self._hp[gi][:1]
        todo = [p for p in params if not self.state[p]]
        if todo:
            flat = torch.zeros(sum((p.numel() + 3) // 4 * 4 for p in todo), dtype=torch.float32, device=todo[0].device)
            off = 0
            for p in todo:
                self.state[p]["momentum_buffer"] = flat[off: off + p.numel()].view_as(p)
                off += (p.numel() + 3) // 4 * 4
        shadows = None
        if cuda:  # the bf16 copies that are up to date stay so; others are cast by the next forward
            shadows = [getattr(p, _SHADOW, None) for p in params]
            shadows = [sh if sh is not None and sh.shape == p.shape and getattr(p, _SHADOW_VER, None) == p._version
                       else None for p, sh in zip(params, shadows)]
        muon_ops.muon_update_(params, [p.grad.float() for p in params],
                              [self.state[p]["momentum_buffer"] for p in params], lr=lr, momentum=group["momentum"],
                              nesterov=group["nesterov"], weight_decay=group["weight_decay"], steps=group["ns_steps"],
                              coefficients=group["ns_coefficients"], rms=group["rms"], shadows=shadows,
                              inv_scale=inv_scale, skip=skip, precise=group.get("precise", False))
        if cuda:
            for p, sh in zip(params, shadows):
                if sh is not None:  # written with the weights: of their new version
                    setattr(p, _SHADOW_VER, p._version)
            self._ensure_grad_buffers()


def _refuse_flat_shards(params) -> None:
    if any(getattr(p, "_md_fsdp", False) for p in params):
        raise ValueError("Muon orthogonalises whole matrices, FSDP keeps flat shards of them: use DDP, or FusedAdamW "
                         "for these parameters")


def muon_groups(model: torch.nn.Module, weight_decay: float | None = None) -> list[dict]:
    """``model``'s parameters as Muon's groups: the matrices of its blocks, and (``orthogonal=False``) the
    embeddings, the LM head and everything that is not a matrix.  ``weight_decay`` applies to matrices
    of both groups; biases and norms, a group of their own, then take none.  A model sharded by FSDP is
    refused."""
    _refuse_flat_shards(model.parameters())
    hidden, tables, small = [], [], []
    for name, p in model.named_parameters():
        if not p.requires_grad:
            continue
        outer = any(part in ("wte", "wpe", "head", "embedding", "lm_head") for part in name.split("."))
        (small if p.dim() < 2 else tables if outer or p.dim() != 2 else hidden).append(p)
    groups = [dict(params=hidden, orthogonal=True), dict(params=tables, orthogonal=False),
              dict(params=small, orthogonal=False)]
    if weight_decay is not None:
        groups[0]["weight_decay"] = groups[1]["weight_decay"] = weight_decay
        groups[2]["weight_decay"] = 0.0
    return [g for g in groups if g["params"]]
