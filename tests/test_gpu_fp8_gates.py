"""Gates over their whole range, from blocks of ordinary values to blocks that the gate alone makes nothing of, against 64 bits.

The bound of one value y = g s(z) u (s the sigmoid): the exponential within two steps (4 U32; the quotient passes no more on), a product, a
sum, a quotient and the product with u, a rounding each: 8 U32. gelu's z: three roundings in the cubic term, one in the
sum, two in the factor, all of one sign: 6 U32 of z, which the sigmoid passes on |z| (1 - s(z)) fold. The exponential of -|z| may be
zero where it is below f32's normal range, 2^-126 (2^-125 with its error); what is g s(z) before the product with u is known to a
step of the subnormals."""
import numpy as np
import pytest
import torch

from tests import fp8_plain as P

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gated(g, u, gelu):
    """(y, its error in the kernel's arithmetic), float64."""
    z = 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3) if gelu else g
    y = g * torch.sigmoid(z) * u
    e = 8 * P.U32 + (6 * P.U32 * z.abs() * torch.sigmoid(-z) if gelu else 0)
    none = (z < 0) & (torch.exp(-z.abs()) < 2.0 ** -125)
    return y, torch.where(none, y.abs(), e * y.abs() + u.abs() * 2.0 ** -149)


def check(a8, asc, y, err, M):
    """The rows and scales of values y known up to err; no block may have its largest value within err of 2^-100."""
    F = y.shape[1]
    p = torch.zeros((2, M, P.up(F, 128)), dtype=torch.float64)
    p[0, :, :F], p[1, :, :F] = y, err
    top, terr = (v.view(M, -1, 128) for v in p)
    top, terr = top.abs().amax(2), terr.amax(2)
    live = top >= P.TINY
    assert bool(((top - P.TINY).abs() > 2 * terr).all())
    asc, q = asc.cpu().double()[:, :M].T, P.value(a8.cpu())[:M]
    wide = lambda v: v[:, :, None].expand(-1, -1, 128).reshape(M, -1)  # noqa: E731
    assert not asc[~live].any() and not q[~wide(live)].any()
    off = (asc - top / 448).abs()
    assert bool((off <= terr / 448 + 2 * P.U32 * top / 448)[live].all()), float((off / top * 448)[live].max())
    s = torch.where(live, 448 / torch.where(live, top, 1.0), 0.0)
    v = p[0] * wide(s)
    e = p[1] * wide(s) + v.abs() * (wide(terr / torch.where(live, top, 1.0)) + 4 * P.U32)
    assert P.near_e4m3(q, v, 1.1 * e)  # (1.1: an error near a border is a step there)


SILU = [(-90.0, 1e5), (-90.0, 1.0), (-84.0, 1e5), (-86.0, 1e6), (-82.0, 1e6), (-60.0, 1.0), (-200.0, 1e30), (-3e38, 1.0), (-1e20, 1e6),
        (-1e30, 1e8), (3e38, 0.5), (1e20, -1e10), (90.0, 1.0), (-1e-30, 1e5)]
GELU = [(-12.0, 1e5), (-20.0, 1e30), (-8.0, 1e5), (-9.9, 1e8), (-5.0, 1.0), (-1e10, 1e10), (-3e38, 1.0), (3e38, -0.5), (1e15, 1.0), (20.0, 1.0)]


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("gelu,pairs", [(False, SILU), (True, GELU)])
def test_blocks_of_far_gates(qm, dev, gelu, pairs, x_type):
    """A block of one gate and one factor each."""
    M, F = len(pairs), 256
    gu = torch.zeros((M, 2 * F))
    for m, (g, u) in enumerate(pairs):
        gu[m, :F], gu[m, F:] = g, u
    gu[:, 128:F] = 1.0  # (a block beside it)
    gu[:, F + 128:] = 1.0
    gu = gu.to(x_type)
    a8, asc = qm.swiglu_fp8(gu.to(dev), F, gelu=gelu)
    check(a8, asc, *gated(gu.double()[:, :F], gu.double()[:, F:], gelu), M)


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("M,F,scale", [(3, 17408, 3.0), (40, 1000, 0.01), (7, 640, 30.0), (260, 512, 1.0)])
def test_every_value_within_its_own_bound(qm, dev, M, F, scale, x_type, gelu):
    """Relative to the value itself, also where the sigmoid is nearly nothing."""
    rng = np.random.default_rng(F + M)
    gu = torch.from_numpy((rng.standard_normal((M, 2 * F)) * scale).astype(np.float32))
    gu[:, F:] /= scale
    if M == 7:  # every block negative: its scale is that of small values
        gu[:, :F] = -gu[:, :F].abs().clamp(max=9.0 if gelu else 80.0)
    gu = gu.to(x_type)
    a8, asc = qm.swiglu_fp8(gu.to(dev), F, gelu=gelu, M_stride=P.up(M, 16))
    check(a8, asc, *gated(gu.double()[:, :F], gu.double()[:, F:], gelu), M)
    assert not a8.cpu().view(torch.uint8)[M:].any() and not a8.cpu().view(torch.uint8)[:, F:].any() and not asc.cpu()[:, M:].any()
