"""Rotary positions against complex rotation in 64 bits.

Tolerance of an element: half a unit in the last place of the result's type, plus the fp32
arithmetic in front of it (two products, one sum, a rounded table entry: under eight fp32 roundings
of |a| + |b|), plus half the smallest subnormal."""

from __future__ import annotations

import pytest
import torch

import minidist as md
from minidist.ops import _native as nat
from minidist.ops import rotary as R

HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _reference(x, angle, interleaved, factor=1.0, inverse=False):
    """``angle [.., S, pairs]`` in 64 bits."""
    y = x.detach().double().clone()
    r = 2 * angle.shape[-1]
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2: r])
    z = torch.complex(a, b) * torch.polar(torch.full_like(angle, factor), -angle if inverse else angle).unsqueeze(-2)
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        y[..., : r // 2], y[..., r // 2: r] = z.real, z.imag
    return y


def _close(y, x, ref, angle_dim, interleaved):
    r = 2 * angle_dim
    f = x.detach().double().abs()
    size = f.clone()
    if interleaved:
        s = f[..., 0:r:2] + f[..., 1:r:2]
        size[..., 0:r:2], size[..., 1:r:2] = s, s
    else:
        s = f[..., : r // 2] + f[..., r // 2: r]
        size[..., : r // 2], size[..., r // 2: r] = s, s
    bound = HALF_ULP[y.dtype] * ref.abs() + 8 * 2.0**-24 * size + TINY[y.dtype]
    assert y.shape == ref.shape
    assert bool(((y.double() - ref).abs() <= bound).all()), float(((y.double() - ref).abs() - bound).max())


def _angle(positions, r, base=10000.0):
    f = base ** (-2.0 * torch.arange(r // 2, dtype=torch.float64, device=positions.device) / r)
    return positions.double()[..., None] * f


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,Hk,D,r", [(2, 7, 4, 4, 64, 64), (1, 1, 3, 1, 128, 64), (3, 5, 2, 2, 80, 40),
                                          (1, 33, 5, 1, 96, 50), (1, 3, 1, 1, 7, 6), (2, 2, 1, 1, 2, 2),
                                          (1, 700, 12, 12, 64, 32), (300, 1, 32, 8, 128, 128)])
def test_against_complex(device, dtype, interleaved, B, S, H, Hk, D, r):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(B, S, H, D, generator=g).to(device, dtype).requires_grad_(True)
    k = torch.randn(B, S, Hk, D, generator=g).to(device, dtype).requires_grad_(True)
    pos = torch.randint(0, 5000, (B, S), generator=g).to(device)
    table = md.rotary_table(r, 5000, device=device)
    y, z = md.apply_rotary(q, k, table, pos, interleaved=interleaved)
    assert y.is_contiguous() and z.is_contiguous()
    angle = _angle(pos, r)
    _close(y, q, _reference(q, angle, interleaved), r // 2, interleaved)
    _close(z, k, _reference(k, angle, interleaved), r // 2, interleaved)
    dy, dz = torch.randn(y.shape, generator=g).to(device, dtype), torch.randn(z.shape, generator=g).to(device, dtype)
    dq, dk = torch.autograd.grad((y, z), (q, k), (dy, dz))
    _close(dq, dy, _reference(dy, angle, interleaved, inverse=True), r // 2, interleaved)
    _close(dk, dz, _reference(dz, angle, interleaved, inverse=True), r // 2, interleaved)
    if device == "cuda":
        nat.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """The op is linear in q: a difference over any step equals the gradient's product, up to rounding."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 9, 3, 32, generator=g).to(device).requires_grad_(True)
    step, w = (torch.randn(2, 9, 3, 32, generator=g).to(device) for _ in range(2))
    table = md.rotary_table(24, 16, device=device)

    def f(x):
        return (md.apply_rotary(x, None, table)[0].double() * w.double()).sum()

    (dq,) = torch.autograd.grad(md.apply_rotary(q, None, table)[0], q, w)
    with torch.no_grad():
        slope = (f(q + step) - f(q - step)) / 2
    # 1728 products, each off by a few fp32 roundings of numbers of size 1.
    assert abs(float(slope - (dq.double() * step.double()).sum())) < 1728 * 16 * 2.0**-24


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 0), (0, 3), (2, 4), (4, 8), (8, 16)])
def test_views(device, shift, pad):
    """q and k inside a packed projection with any row padding and start; other orders of the axes."""
    B, S, H, D = 2, 13, 3, 32
    g = torch.Generator().manual_seed(2)
    buf = torch.randn(B * S * (3 * H * D + pad) + shift, generator=g).to(device, torch.bfloat16)
    packed = buf[shift:].as_strided((B, S, H, 3, D), (S * (3 * H * D + pad), 3 * H * D + pad, 3 * D, D, 1),
                                    buf.storage_offset() + shift)
    table = md.rotary_table(32, S, device=device)
    q, k = packed[:, :, :, 0], packed[:, :, :, 1]
    angle = _angle(torch.arange(S, device=device), 32)
    y, z = md.apply_rotary(q, k, table)
    _close(y, q, _reference(q, angle, False), 16, False)
    _close(z, k, _reference(k, angle, False), 16, False)
    t = q.contiguous().transpose(1, 2).contiguous().transpose(1, 2)  # heads before tokens in memory
    assert torch.equal(md.apply_rotary(t, None, table)[0], y)
    odd = torch.randn(B, S, H, 2 * D, generator=g).to(device, torch.bfloat16)[..., ::2]  # channels two apart
    _close(md.apply_rotary(odd, None, table)[0], odd, _reference(odd, angle, False), 16, False)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_in_place(device):
    B, S, H, D = 2, 11, 3, 64
    g = torch.Generator().manual_seed(3)
    buf = torch.randn(B * S, 3 * H * D + 8, generator=g).to(device, torch.bfloat16)
    qkv, before = buf[:, : 3 * H * D], buf.clone()
    table = md.rotary_table(48, S + 2, device=device)
    R.rotate_packed_(qkv, H, table, batch=B)
    old, new = (t[:, : 3 * H * D].reshape(B, S, H, 3, D) for t in (before, buf))
    y, z = md.apply_rotary(old[..., 0, :], old[..., 1, :], table)
    assert torch.equal(new[..., 0, :], y) and torch.equal(new[..., 1, :], z)
    assert torch.equal(new[..., 2, :], old[..., 2, :]) and torch.equal(buf[:, 3 * H * D:], before[:, 3 * H * D:])
    R.rotate_packed_(qkv, H, table, batch=B, inverse=True)  # and back, up to two roundings
    back = buf[:, : 3 * H * D].double() - before[:, : 3 * H * D].double()
    # each rounding moves a channel by half a unit of a number no larger than the pair
    assert float(back.abs().max()) <= 3 * 2.0**-8 * 2 * float(before.abs().max())


@pytest.mark.parametrize("device", DEVICES)
def test_positions_forms(device):
    q = torch.randn(2, 6, 2, 16).to(device)
    table = md.rotary_table(16, 40, device=device)
    row = torch.arange(30, 36, device=device)
    y = md.apply_rotary(q, None, table, row)[0]
    for pos in (row.int(), row.expand(2, 6), row.int()[None].repeat(2, 1), torch.stack([row, row], 1)[:, 0]):
        assert torch.equal(md.apply_rotary(q, None, table, pos)[0], y)
    assert torch.equal(md.apply_rotary(q, None, table)[0],
                       md.apply_rotary(q, None, table, torch.arange(6, device=device))[0])
    assert md.apply_rotary(q[:, :0], None, table)[0].shape == (2, 0, 2, 16)
    assert md.apply_rotary(q[:0], q[:0], table)[1].shape == (0, 6, 2, 16)


def test_tables():
    r, n = 32, 64
    i = torch.arange(r // 2, dtype=torch.float64)
    inv = 10000.0 ** (-2 * i / r)
    pos = torch.arange(n, dtype=torch.float64)[:, None]

    def same(table, freq, factor=1.0):
        ref = torch.stack([(pos * freq).cos(), (pos * freq).sin()], -1) * factor
        # fp32 rounding of a 64-bit value of size up to the factor
        assert float((table.double() - ref).abs().max()) <= 2.0**-24 * factor

    same(md.rotary_table(r, n), inv)
    same(md.rotary_table(r, n, scaling=md.RotaryScaling("linear", 8.0)), inv / 8)
    same(md.rotary_table(r, n, scaling=md.RotaryScaling("ntk", 8.0)), (10000.0 * 8 ** (r / (r - 2))) ** (-2 * i / r))
    yarn = md.rotary_table(r, n, scaling=md.RotaryScaling("yarn", 8.0, original_positions=4096))
    factor = 0.1 * torch.log(torch.tensor(8.0, dtype=torch.float64)).item() + 1
    # The fastest pair turns 652 times in 4096 positions: kept; the slowest 0.1 times: divided.
    same(yarn[:, :1], inv[:1], factor)
    same(yarn[:, -1:], inv[-1:] / 8, factor)
    first = torch.atan2(yarn[1, :, 1], yarn[1, :, 0]).double()  # the frequencies themselves
    assert bool((first <= inv * (1 + 1e-6)).all()) and bool((first >= inv / 8 * (1 - 1e-6)).all())


@pytest.mark.gpu
def test_position_outside_the_table_is_reported():
    nat.check_status()
    q = torch.randn(1, 3, 2, 16, device="cuda")
    table = md.rotary_table(8, 10, device="cuda")
    y = md.apply_rotary(q, None, table, torch.tensor([0, 10, -1], device="cuda"))[0]
    assert torch.equal(y[:, :1], q[:, :1]) and torch.equal(y[..., 8:], q[..., 8:])
    assert bool(y[:, 1:, :, :8].isnan().all())
    with pytest.raises(nat.NativeError, match="bad kernel argument"):
        nat.check_status()


@pytest.mark.gpu
def test_other_stream():
    table = md.rotary_table(64, 512, device="cuda")
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        big = big @ big * 1e-2  # keeps the default stream busy: the call below must not wait for it or overtake
    q = torch.randn(8, 512, 4, 64, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q2 = q * 2
        y = md.apply_rotary(q2, None, table)[0]
    torch.cuda.current_stream().wait_stream(side)
    _close(y, q2, _reference(q2, _angle(torch.arange(512, device="cuda"), 64), False), 32, False)


def test_refusals():
    q = torch.zeros(1, 4, 2, 16)
    table = md.rotary_table(16, 8)
    for bad in (
        lambda: md.apply_rotary(q[0], None, table),
        lambda: md.apply_rotary(q, torch.zeros(1, 5, 2, 16), table),
        lambda: md.apply_rotary(q, torch.zeros(1, 4, 2, 8), table),
        lambda: md.apply_rotary(q, q.half(), table),
        lambda: md.apply_rotary(q.double(), None, table),
        lambda: md.apply_rotary(q, None, md.rotary_table(18, 8)),
        lambda: md.apply_rotary(q, None, table.double()),
        lambda: md.apply_rotary(q, None, table[:, ::2]),
        lambda: md.apply_rotary(q, None, table[:3]),
        lambda: md.apply_rotary(q, None, table, torch.zeros(3, dtype=torch.long)),
        lambda: md.apply_rotary(q, None, table, torch.zeros(4)),
        lambda: md.rotary_table(15, 8),
        lambda: md.rotary_table(0, 8),
        lambda: md.rotary_table(16, -1),
        lambda: md.RotaryScaling("cubic", 2.0),
        lambda: md.RotaryScaling("linear", 0.5),
    ):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(IndexError):
        md.apply_rotary(q, None, table, torch.tensor([0, 1, 2, 8]))
