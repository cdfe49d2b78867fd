"""How many matrices a call of the kernels takes, and what memory it needs for them."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import muon as M

pytestmark = pytest.mark.gpu


def _peak(fn):
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    fn()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - base


@pytest.mark.parametrize("precise", [False, True])
def test_workspace_is_bounded(monkeypatch, precise):
    w, g, m = ([torch.randn(640, 384, device="cuda") for _ in range(20)] for _ in range(3))
    u = torch.stack(g)
    one = nat.lib().md_muon_workspace(1, 640, 384, precise)
    twins = [[t.clone() for t in x] for x in (w, m)]
    free = _peak(lambda: M.muon_update_(w, g, m, lr=0.1, precise=precise))
    whole = md.orthogonalize(u, precise=True)
    monkeypatch.setattr(M, "_WORKSPACE", 3 * one + 100)
    bound = _peak(lambda: M.muon_update_(twins[0], g, twins[1], lr=0.1, precise=precise))
    assert free > 15 * one and bound < 4 * one + (1 << 20)
    for a, b in zip(m, twins[1]):
        assert torch.equal(a, b)
    for a, b in zip(w, twins[0]):  # (other tiles, perhaps: other roundings of the same scheme)
        assert float((a - b).norm()) < 1.2e-2 * 0.1 * 0.2 * 640**0.5 * 384**0.5
    parts = md.orthogonalize(u, precise=True)
    assert float((whole - parts).norm() / whole.norm()) < 1.2e-5
    monkeypatch.setattr(M, "_WORKSPACE", 1)  # one matrix is always taken
    assert float((whole - md.orthogonalize(u, precise=True)).norm() / whole.norm()) < 1.2e-5
    nat.check_status()
