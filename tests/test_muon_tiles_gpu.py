"""The Muon step through every tile size, with several tiles per SM and edges inside them.

Tolerances come from the scheme itself: ``_scheme`` makes, in 64 bits, the roundings that the kernels make
by design (X as two fp16 parts, the products' operands one, each at 2^12 times its value).  The kernels
round the same numbers, but other ones once a rounding has gone the other way; sums of ten thousand and
more independent errors of one size differ by a few per cent, so 1.3 times the scheme's error is a
generous limit.  1e-4 is added for the accumulators, which truncate (2^-23 of a partial sum each time,
over up to 150 additions: 2e-5 in the worst case, carried through five steps)."""

from __future__ import annotations

import math

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import muon as M

DEV = pytest.mark.gpu
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


def _half(x):
    return (x * 4096).half().double() / 4096


def _scheme(u, low=True):
    """Exact but for the kernels' roundings; ``low=False`` leaves out X's low part (a mistake)."""
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    x = x if x.shape[-2] <= x.shape[-1] else x.mT
    for _ in range(5):
        high = _half(x)
        whole = high + _half(x - high) if low else high
        g = _half(high @ high.mT)
        x = A * whole + _half(B * g + C * g @ g) @ high
    return x if u.shape[-2] <= u.shape[-1] else x.mT


def _off(x, ref):
    return float((x.double() - ref).norm() / ref.norm())


def _limit(u):
    return 1.3 * _off(_scheme(u), _exact(u)) + 1e-4


def _matrices(count, rows, cols, device, decay=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(count, rows, cols, generator=g)
    if decay:  # a few strong directions over a floor: the floor's singular values are what low parts keep
        u = u * 0.05 + torch.randn(count, rows, 3, generator=g) @ torch.randn(count, 3, cols, generator=g)
    return u.to(device)


def test_the_limit_tells_the_low_part_from_its_absence():
    for rows, cols in ((96, 200), (200, 96), (130, 131)):
        u = _matrices(1, rows, cols, "cpu", decay=True)[0]
        assert _off(_scheme(u, low=False), _exact(u)) > 1.5 * _limit(u)
        assert _limit(u) < 6e-3


SHAPES = [(40, 300, 500), (40, 500, 300), (20, 301, 517), (20, 517, 301), (3, 768, 2304), (3, 2304, 768), (64, 40, 96),
          (1, 1, 33), (2, 33, 1)]


def _start(count, rows, cols, shift, decay=False):
    """Weights, gradients, momenta, copies; each ``shift`` elements into its memory."""
    out = []
    for i, scale in enumerate((0.05, 1e-3, 3e-3)):
        flat = torch.empty(count, rows * cols + 5, device="cuda")
        t = flat[:, shift: shift + rows * cols].view(count, rows, cols)
        t.copy_(_matrices(count, rows, cols, "cuda", decay=decay and i > 0, seed=7 * i) * scale)
        out.append(list(t.unbind()))
    copies = torch.empty(count, rows * cols + 5, dtype=torch.bfloat16, device="cuda")
    copies = list(copies[:, shift: shift + rows * cols].view(count, rows, cols).unbind())
    return (*out, copies)


def _check_step(w, g, m, copies, limit_of, tile, precise, shift):
    rows, cols = w[0].shape
    lr, mu, wd = 0.02, 0.9, 0.1
    rate = lr * 0.2 * math.sqrt(max(rows, cols))
    new_m = [mu * b.double() + a.double() for a, b in zip(g, m)]
    u = [a.double() + mu * b for a, b in zip(g, new_m)]
    old = [t.clone() for t in w]
    shadows = [c if i % 3 else None for i, c in enumerate(copies)]
    M._step_cuda(w, g, m, shadows, lr, mu, True, wd, 5, M.COEFFICIENTS, 1e-7, 0.2, None, None, precise, tile)
    nat.check_status()
    for i in range(len(w)):
        ref = _exact(u[i])
        off = float((w[i].double() - ((1 - lr * wd) * old[i].double() - rate * ref)).norm())
        assert off < limit_of(u[i]) * rate * float(ref.norm()) + 3 * 2.0**-24 * float(old[i].double().norm()), i
        # two fp32 roundings of the momentum
        assert float((m[i].double() - new_m[i]).abs().max()) < 2 * 2.0**-24 * float(new_m[i].abs().max()) * 2
        if shadows[i] is not None:
            assert torch.equal(shadows[i], w[i].bfloat16())


@DEV
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("shift", [0, 1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_step(shape, shift, tile):
    if shift and shape[0] == 3:
        pytest.skip("one start is enough for the large ones")
    small = min(shape[1:]) < 33  # too few numbers for the size of their errors to be a size: the worst rounding
    _check_step(*_start(*shape, shift), (lambda u: 1.2e-2) if small else _limit, tile, False, shift)


@DEV
@pytest.mark.parametrize("tile", [1, 2, 3])
@pytest.mark.parametrize("shape", [(40, 300, 500), (40, 500, 300), (3, 768, 2304)])
def test_step_of_a_decaying_spectrum(shape, tile):
    def limit(u):
        assert _off(_scheme(u, low=False), _exact(u)) > 1.5 * _limit(u)  # it would be seen
        return _limit(u)

    _check_step(*_start(*shape, 0, decay=True), limit, tile, False, 0)


@DEV
@pytest.mark.parametrize("tile", [0, 1, 3])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("shape", [(40, 300, 500), (40, 500, 300), (20, 301, 517), (1, 203, 1001), (3, 768, 2304)])
def test_precise_step(shape, shift, tile):
    """Three products: as far off as fp32's own, or 6e-6 (22 bits of what single products make 11)."""
    def limit(u):
        return max(6e-6, 2 * _off(M._orthogonal_cpu(u.float(), 5, M.COEFFICIENTS, 1e-7), _exact(u)))

    _check_step(*_start(*shape, shift), limit, tile, True, shift)


@DEV
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("shape", [(30, 300, 500), (20, 517, 301), (2, 1030, 1100), (1, 200, 4200)])
def test_bfloat16_answers(shape, tile):
    """Off by the scheme's error and the answer's own rounding (2^-9 at most)."""
    u = _matrices(*shape, "cuda", decay=True).bfloat16()
    x = M._orthogonalize_cuda(u, 5, M.COEFFICIENTS, 1e-7, tile=tile)
    nat.check_status()
    for i in range(shape[0]):
        assert _off(x[i], _exact(u[i])) < math.hypot(_limit(u[i]), 2.0**-9), i


@DEV
@pytest.mark.parametrize("shape", [(300, 900), (900, 300), (4, 96, 257), (768, 2304)])
def test_precise_bfloat16_answers_are_rounded_exact_ones(shape):
    u = torch.randn(*shape, generator=torch.Generator().manual_seed(3)).to("cuda", torch.bfloat16)
    x, ref = md.orthogonalize(u, precise=True), _exact(u)
    nat.check_status()
    assert _off(x, ref) < 2.0**-9
    # An error of 6e-6 of the entries' size moves an entry over a rounding boundary in 6e-6 * 2^8 of the
    # cases times that size over the entry's own: 5 on average over entries above 1.5e-3 of it, which
    # all but 1.2e-3 of them are.
    assert float((x != ref.bfloat16()).double().mean()) < 6e-6 * 2**8 * 5 + 1.2e-3
    assert not torch.equal(x, md.orthogonalize(u))
    assert torch.equal(md.orthogonalize(u.float(), precise=True), md.orthogonalize(u.float()))
