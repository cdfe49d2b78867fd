"""What ``muon_update_`` refuses of the scalars that its kernels read through a pointer.  Host only:
nothing is launched."""

from __future__ import annotations

import pytest
import torch

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
