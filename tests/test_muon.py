"""Newton-Schulz orthogonalisation and the Muon step against 64 bits.

Tolerances (Frobenius, relative).  Let q be the sum of the sizes of the polynomial's terms, at most
a + 2 |b| + 4 c < 22 for singular values below 1.4, against results near one.  A step rounds X, A and B
once each to 11 bits (2^-12 on average over a binade, random): under sqrt(3) q 2^-12 / sqrt(3) = 5e-3
per step, of which the polynomial's slope carries at most all over; five steps, added as random
errors, stay under 1.2e-2 and, measured against the bf16 rounding of the answer (2^-9), nobody needs
it finer.  Three products keep 22 bits: the same argument gives 1.2e-2 * 2^-11 = 6e-6 for wide
matrices of independent entries, whose smallest singular value is not far below the others; for others
it is compared with what fp32 itself makes of the matrix."""

from __future__ import annotations

import math

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import muon as M

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
ONE_PRODUCT = 1.2e-2
THREE_PRODUCTS = 6e-6
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _exact(u, steps=5, coefficients=M.COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.detach().double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    wide = x.shape[-2] <= x.shape[-1]
    for _ in range(steps):
        g = x @ x.mT if wide else x.mT @ x
        p = b * g + c * g @ g
        x = a * x + (p @ x if wide else x @ p)
    return x


def _off(x, ref):
    return float((x.double() - ref).norm() / ref.norm().clamp(min=1e-300))


def _matrix(*shape, seed=0, decay=False):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(*shape, generator=g)
    if decay:  # a few strong directions over a floor
        u = u * 0.05 + torch.randn(*shape[:-1], 3, generator=g) @ torch.randn(*shape[:-2], 3, shape[-1], generator=g)
    return u


SHAPES = [(1, 1), (1, 9), (9, 1), (8, 8), (5, 64), (129, 127), (64, 300), (300, 64), (128, 128), (256, 512),
          (512, 256), (257, 259), (130, 1000), (1000, 130), (768, 768), (203, 1001)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_orthogonalize(device, dtype, shape):
    u = _matrix(*shape).to(device, dtype)
    x = md.orthogonalize(u)
    ref = _exact(u)
    assert x.dtype == dtype and x.shape == u.shape
    if dtype == torch.bfloat16:
        assert _off(x, ref) < (ONE_PRODUCT**2 + HALF_ULP[dtype]**2) ** 0.5
    else:
        # square ones: as far as fp32 products are off, or twice that
        plain = _off(M._orthogonal_cpu(u.cpu(), 5, M.COEFFICIENTS, 1e-7), ref.cpu())
        assert _off(x, ref) < max(THREE_PRODUCTS, 2 * plain) + HALF_ULP[dtype]
    if device == "cuda":
        nat.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("shape", [(3, 70, 40), (2, 256, 256), (2, 300, 700), (3, 700, 300), (1, 1100, 1030),
                                   (70, 40, 24), (1, 100, 1100), (2, 2100, 130), (1, 200, 4200)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tiles_and_batches(tile, shape, dtype):
    """Every tile size, and the choice, at sizes that end inside a tile, with K shared by a cluster, several
    tiles per SM, more matrices than a call takes."""
    u = _matrix(*shape, seed=1, decay=dtype == torch.bfloat16).to("cuda", dtype)
    x = M._orthogonalize_cuda(u, 5, M.COEFFICIENTS, 1e-7, tile=tile)
    nat.check_status()
    ref = _exact(u)
    for i in range(shape[0]):
        plain = _off(M._orthogonal_cpu(u[i], 5, M.COEFFICIENTS, 1e-7), ref[i])
        limit = ONE_PRODUCT + 2.0**-8 if dtype == torch.bfloat16 else max(THREE_PRODUCTS, 2 * plain)
        assert _off(x[i], ref[i]) < limit, i
    assert torch.equal(x, M._orthogonalize_cuda(u, 5, M.COEFFICIENTS, 1e-7, tile=tile))  # bit for bit


@pytest.mark.parametrize("device", DEVICES)
def test_forms(device):
    u = _matrix(2, 3, 40, 24).to(device)
    x = md.orthogonalize(u)
    assert x.shape == u.shape
    for i in range(2):
        for j in range(3):
            assert _off(x[i, j], _exact(u[i, j])) < 1e-4
    t = md.orthogonalize(u[0, 0].t())  # a transposed view
    assert _off(t, _exact(u[0, 0].t())) < 1e-4
    wide = _matrix(40, 80).to(device)[:, ::2]  # columns two apart
    assert _off(md.orthogonalize(wide), _exact(wide)) < 1e-4
    for steps, co in ((1, M.COEFFICIENTS), (12, (1.5, -0.5, 0.0)), (8, (15 / 8, -10 / 8, 3 / 8))):
        v = _matrix(30, 90, seed=3).to(device)
        x = md.orthogonalize(v, steps=steps, coefficients=co)
        assert _off(x, _exact(v, steps, co)) < 1e-4
    # the classical coefficients converge: X X^T = I
    assert float((x @ x.t() - torch.eye(30, device=device)).abs().max()) < 1e-2
    assert md.orthogonalize(torch.zeros(0, 5, device=device)).shape == (0, 5)
    assert bool((md.orthogonalize(torch.zeros(6, 5, device=device)) == 0).all())
    for scale in (1e-12, 1e12):  # the norm takes out any scale (above eps)
        v = _matrix(33, 70).to(device) * scale
        assert _off(md.orthogonalize(v, eps=0.0), _exact(v, eps=0.0)) < 1e-4
    v[0, 0] = float("nan")
    assert bool(md.orthogonalize(v).isnan().all())


def _step_reference(w, g, m, lr, mu, nesterov, wd, rms=0.2):
    w, g, m = w.double(), g.double(), m.double()
    m = mu * m + g
    u = g + mu * m if nesterov else m
    x = _exact(u)
    return (1 - lr * wd) * w - lr * rms * math.sqrt(max(w.shape)) * x, m, lr * rms * math.sqrt(max(w.shape)) * x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(device, nesterov):
    shapes = [(40, 24), (24, 40), (40, 24), (129, 300), (1, 7), (64, 64)]
    new = lambda seed, s=1.0: [(_matrix(*sh, seed=seed + i) * s).to(device) for i, sh in enumerate(shapes)]  # noqa: E731
    w, g, m = new(0), new(10, 1e-3), new(20, 5e-3)
    g[1] = g[1].t().contiguous().t()  # a gradient in another order
    shadows = [torch.zeros(sh, dtype=torch.bfloat16, device=device) if i % 2 else None for i, sh in enumerate(shapes)]
    hp = dict(lr=0.02, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
    want = [_step_reference(*t, 0.02, 0.9, nesterov, 0.1) for t in zip(w, g, m)]
    before = [t.clone() for t in w]
    md.ops.muon.muon_update_(w, g, m, shadows=shadows, **hp)
    for i, (rw, rm, dx) in enumerate(want):
        limit = ONE_PRODUCT if device == "cuda" else 1e-4
        # the weights are off by what their update is, plus three fp32 roundings
        assert float((w[i].double() - rw).norm()) < limit * float(dx.norm()) + 3 * 2.0**-24 * float(rw.norm()), i
        assert _off(m[i], rm) < 3 * 2.0**-24
        assert not torch.equal(w[i], before[i])
        if shadows[i] is not None:
            assert torch.equal(shadows[i], w[i].bfloat16())


@pytest.mark.gpu
def test_step_device_learning_rate_scale_and_skip():
    w = [_matrix(96, 200, seed=i).cuda() for i in range(3)]
    g = [_matrix(96, 200, seed=5 + i).cuda() for i in range(3)]
    m = [torch.zeros_like(t) for t in w]
    copies = [[t.clone() for t in x] for x in (w, g, m)]
    M.muon_update_(w, g, m, lr=0.01, weight_decay=0.1)
    other = [[t.clone() for t in x] for x in copies]
    scaled = [t * 1024 for t in other[1]]
    M.muon_update_(other[0], scaled, other[2], lr=torch.tensor([0.01], device="cuda"), weight_decay=0.1,
                   inv_scale=torch.tensor([1 / 1024], device="cuda"), skip=torch.zeros(1, device="cuda"))
    for a, b in zip(w + m, other[0] + other[2]):
        assert _off(a, b.double()) < 1e-6
    third = [[t.clone() for t in x] for x in copies]
    M.muon_update_(*third, lr=0.01, skip=torch.ones(1, device="cuda"))
    assert all(torch.equal(a, b) for x, y in zip(third, copies) for a, b in zip(x, y))
    nat.check_status()


@pytest.mark.gpu
def test_many_matrices_and_other_stream():
    w = [_matrix(32, 48, seed=i).cuda() for i in range(130)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = [t * 0.5 for t in w]
        m = [torch.zeros_like(t) for t in w]
        ref = [_step_reference(a, b, c, 0.1, 0.95, True, 0.0) for a, b, c in zip(w, g, m)]
        M.muon_update_(w, g, m, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    for a, (b, _, dx) in zip(w, ref):
        assert float((a.double() - b).norm()) < ONE_PRODUCT * float(dx.norm()) + 1e-6


def test_refusals():
    w, g, m = torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6)
    for bad in (
        lambda: md.orthogonalize(torch.zeros(5)),
        lambda: md.orthogonalize(w.double()),
        lambda: md.orthogonalize(w, steps=0),
        lambda: md.orthogonalize(w, coefficients=(1.0, 2.0)),
        lambda: md.orthogonalize(w, eps=-1.0),
        lambda: M.muon_update_([w], [g], [], lr=0.1),
        lambda: M.muon_update_([w[0]], [g[0]], [m[0]], lr=0.1),
        lambda: M.muon_update_([w.t()], [g.t()], [m.t()], lr=0.1),
        lambda: M.muon_update_([w.half()], [g], [m], lr=0.1),
        lambda: M.muon_update_([w], [g[:2]], [m], lr=0.1),
        lambda: M.muon_update_([w], [g.half()], [m], lr=0.1),
        lambda: M.muon_update_([w], [g], [m.double()], lr=0.1),
        lambda: M.muon_update_([w], [g], [m], lr=0.1, shadows=[w]),
    ):
        with pytest.raises((ValueError, TypeError)):
            bad()
