"""What ``muon_update_`` refuses of the scalars that its kernels read through a pointer.  Host only:
nothing is launched."""

from __future__ import annotations

import pytest
import torch

from minidist.ops import muon as M


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
