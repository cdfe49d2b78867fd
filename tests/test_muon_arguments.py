"""What ``muon_update_`` refuses of the scalars that its kernels read through a pointer.  Host only:
nothing is launched."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import muon as M
from minidist.optim import FusedAdamW, Muon


def _state():
    return [[torch.full((4, 6), v)] for v in (1.0, 2.0, 3.0)]


@pytest.mark.parametrize("name", ["inv_scale", "skip", "lr"])
@pytest.mark.parametrize("bad", [torch.ones(1, dtype=torch.float64), torch.ones(1, dtype=torch.int32),
                                 torch.ones(1, dtype=torch.bool), torch.ones(2), torch.ones(0),
                                 torch.ones(1, device="meta")])
def test_scalar_refusals(name, bad):
    w, g, m = _state()
    with pytest.raises(ValueError, match=name):
        M.muon_update_(w, g, m, **{"lr": 0.1, name: bad})
    assert all(torch.equal(a[0], b[0]) for a, b in zip((w, g, m), _state()))


def test_scalars_have_to_be_where_the_matrices_are():
    for device in ("cuda:0", "cuda:1"):
        with pytest.raises(ValueError, match="skip"):
            M._check_scalar(torch.ones(1), "skip", torch.device(device))
    # One flag cannot serve two devices; the first device's matrices stay as they were.
    (w,), (g,), (m,) = _state()
    far = [torch.empty(4, 6, device="meta") for _ in range(3)]
    for order in (1, -1):
        with pytest.raises(ValueError, match="skip"):
            M.muon_update_([w, far[0]][::order], [g, far[1]][::order], [m, far[2]][::order], lr=0.1,
                           skip=torch.zeros(1))
    assert torch.equal(w, torch.full((4, 6), 1.0)) and torch.equal(m, torch.full((4, 6), 3.0))


def test_scalars_that_are_taken():
    for shape in ((), (1,), (1, 1)):
        w, g, m = _state()
        M.muon_update_(w, g, m, lr=torch.full(shape, 0.1), inv_scale=torch.full(shape, 0.5), skip=torch.zeros(shape))
        v, h, n = _state()
        M.muon_update_(v, [h[0] * 0.5], n, lr=0.1)
        assert torch.equal(m[0], n[0]) and float((w[0] - v[0]).abs().max()) <= 2.0**-22
        M.muon_update_(w, g, m, lr=0.1, skip=torch.ones(shape))
        assert torch.equal(m[0], n[0])


class _OnDevice(torch.nn.Parameter):
    """A CPU parameter that says it is on a GPU, for checks that come before any launch."""

    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda:0"))


@pytest.mark.parametrize("cls", [FusedAdamW, Muon])
def test_optimizers_refuse_scalars_elsewhere(cls):
    """Groups whose update is AdamW's kernel read the same two pointers."""
    p = torch.nn.Parameter(torch.ones(4))
    opt = cls([p], lr=0.1)
    p.grad = torch.ones(4)
    with pytest.raises(ValueError, match="inv_scale"):
        opt.step(skip=torch.zeros(2))
    assert torch.equal(p, torch.ones(4))
    opt.step(skip=torch.zeros(1), inv_scale=torch.ones(1))
    q = _OnDevice(torch.ones(4))
    opt = cls([torch.nn.Parameter(torch.ones(4))], lr=0.1)
    opt.param_groups[0]["params"] = [q]
    q.grad = torch.ones(4)
    for bad in (torch.zeros(1), torch.zeros(1, dtype=torch.bool), torch.zeros(1, dtype=torch.float64)):
        for name in ("skip", "inv_scale"):
            with pytest.raises(ValueError, match="cuda:0"):
                opt.step(**{name: bad})


def test_coefficients_that_leave_the_operands_range():
    """fp16 operands hold X, A and B up to 15.99: what could pass that is refused, the usual ones are not."""
    for steps, co in ((5, M.COEFFICIENTS), (100, M.COEFFICIENTS), (40, (1.5, -0.5, 0.0)), (40, (15 / 8, -10 / 8, 3 / 8)),
                      (1, (3.0, -3.2, 1.2)), (1, (8.0, -20.0, 13.0))):
        M._check_range(steps, co)
    for steps, co in ((3, (4.5, -1.0, 0.0)), (2, (1.0, 4.0, 0.0)), (1, (1.0, -16.0, 0.0)), (5, (2.0, 0.0, 0.0)),
                      (1, (1.0, float("nan"), 0.0)), (2, (float("inf"), 0.0, 0.0))):
        with pytest.raises(ValueError, match="range"):
            M._check_range(steps, co)


@pytest.mark.gpu
def test_such_coefficients_on_the_gpu():
    u, bad = torch.randn(16, 24, device="cuda"), (2.0, 0.0, 0.0)
    M._check_range(2, bad)
    assert bool(md.orthogonalize(u, steps=2, coefficients=bad).isfinite().all())
    with pytest.raises(ValueError, match="range"):
        md.orthogonalize(u, coefficients=bad)
    w, m = u.clone(), torch.zeros_like(u)
    with pytest.raises(ValueError, match="range"):
        M.muon_update_([w], [u], [m], lr=0.1, coefficients=bad)
    assert torch.equal(w, u) and not m.any()
    x = md.orthogonalize(u, steps=1, coefficients=(8.0, -20.0, 13.0))  # large, but held
    v = u.double() / u.double().norm()
    g = v @ v.t()
    ref = 8 * v + (-20 * g + 13 * g @ g) @ v
    assert float((x.double() - ref).norm() / ref.norm()) < 1e-4
