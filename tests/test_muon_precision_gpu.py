"""fp32 answers are as near to exact as fp32 products would bring them, at every length of the shorter side.

``orthogonalize`` of wide fp32 matrices against 64 bits, beside five steps of fp32 products (CUDA's own, with
their rounding to nearest): at most 1.5 times as far off, above a floor of 1e-6 (sixteen roundings)."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import muon as M

A, B, C = M.COEFFICIENTS


def _exact(u):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    wide = x.shape[-2] <= x.shape[-1]
    for _ in range(5):
        g = x @ x.mT if wide else x.mT @ x
        p = B * g + C * g @ g
        x = A * x + (p @ x if wide else x @ p)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 12, 70])
@pytest.mark.parametrize("rows,cols", [(48, 96), (1317, 63), (54, 297), (73, 461), (116, 54), (65, 2810), (50, 158),
                                       (64, 128), (128, 256), (1000, 127), (129, 300), (16, 40), (200, 800), (520, 130)])
def test_as_near_as_fp32_products(rows, cols, count):
    u = torch.randn(count, rows, cols, generator=torch.Generator().manual_seed(rows)).cuda()
    ref = _exact(u)
    size = ref.norm()
    plain = float((M._orthogonal_cpu(u, 5, M.COEFFICIENTS, 1e-7) - ref).norm() / size)
    own = float((md.orthogonalize(u) - ref).norm() / size)
    nat.check_status()
    assert own < max(1e-6, 1.5 * plain), (own, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [1, 3])
@pytest.mark.parametrize("rows,cols", [(65, 700), (128, 2000), (3000, 100), (33, 4000)])
def test_every_tile(rows, cols, tile):
    """Short and long K in one call, K shared by a cluster, more tiles than SMs."""
    for count in (1, 150):
        u = torch.randn(count, rows, cols, generator=torch.Generator().manual_seed(cols)).cuda()
        ref = _exact(u)
        plain = float((M._orthogonal_cpu(u, 5, M.COEFFICIENTS, 1e-7) - ref).norm() / ref.norm())
        own = M._orthogonalize_cuda(u, 5, M.COEFFICIENTS, 1e-7, tile=tile)
        assert float((own - ref).norm() / ref.norm()) < max(1e-6, 1.5 * plain)
        assert torch.equal(own, M._orthogonalize_cuda(u, 5, M.COEFFICIENTS, 1e-7, tile=tile))
    nat.check_status()
