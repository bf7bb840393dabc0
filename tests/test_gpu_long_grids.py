"""Calls of more work-groups than one grid holds (2^32 threads of a dimension): every row behind that as the ones before."""
import math

import pytest
import torch

from tests import fp8_plain as P

pytestmark = pytest.mark.gpu

ROWS = (1 << 24) + 21  # (a work-group of 256 threads each)


def test_quantized_rows(qm, dev):
    x = torch.randn((ROWS - 4, 1), device=dev).half()
    a8, asc = qm.quantize_fp8(x, M_stride=ROWS)
    want = torch.zeros(ROWS)
    want[:-4] = x[:, 0].float().cpu()
    assert torch.equal(asc[0].cpu(), want.abs() / 448)
    assert torch.equal(a8[:, 0].float().cpu(), torch.sign(want) * 448) and not a8[:, 1:].view(torch.uint8).any()


def test_padding_of_rows_of_two_work_groups(qm, dev):
    """Few tokens in a batch padded to half as many rows: the rest is cleared to its last byte."""
    Ms, K, M = ROWS // 2, 2049, 3
    x = torch.randn((M, K), device=dev)
    a8 = torch.full((Ms, P.up(K, 128)), 0xFF, dtype=torch.uint8, device=dev)
    asc = torch.full((P.up(K, 128) // 128, Ms), -1.0, device=dev)
    qm._call("qmatmul_quantize_fp8", qm._ptr(x), 0, K, M, Ms, K, qm._ptr(a8), qm._ptr(asc), qm._stream(None))
    q, sc = P.quantize32(x.cpu().numpy())
    assert torch.equal(P.value(a8[:M].cpu()), q) and torch.equal(asc[:, :M].cpu(), sc)
    assert not a8[M:].any() and not asc[:, M:].any()


def test_normed_rows(qm, dev):
    x, w = torch.randn((ROWS, 1), device=dev), torch.full((1,), 3.0, device=dev)
    a8, asc, h = qm.rmsnorm_fp8(x, w, 1e-6, want_h=True)
    d = x.double()
    y = 3 * d / torch.sqrt(d * d + 1e-6)
    assert bool(((h.double() - y).abs() <= P.norm_error(1, 1) * y.abs() + 1e-40).all())
    h = torch.where(h[:, 0].abs() >= P.TINY, h[:, 0], 0.0).cpu()
    assert torch.equal(asc[0].cpu(), h.abs() / 448) and torch.equal(a8[:, 0].float().cpu(), torch.sign(h) * 448)


def test_turned_tokens(qm, dev):
    """Four tokens a work-group."""
    T = 4 * ROWS
    x = torch.randn((T, 2), device=dev)
    pos, f = torch.arange(T, dtype=torch.int32, device=dev), torch.tensor([1.0], device=dev)
    q, k = qm.qk_norm_rope(x, 1, 0, 2, pos, f)
    assert k.shape == (T, 0, 2)
    for t in range(0, T, 1 << 24):
        u, v = x[t:t + (1 << 24)].double().unbind(1)
        a = pos[t:t + (1 << 24)].double()
        c, s = torch.cos(a), torch.sin(a)
        e = (4 + math.pi + 3 + 3 + 1) * P.U32 * (u.abs() + v.abs())  # (angle, cosine and sine, products, the result's rounding)
        got = q[t:t + (1 << 24), 0].double()
        assert bool(((got[:, 0] - (u * c - v * s)).abs() <= e).all()) and bool(((got[:, 1] - (v * c + u * s)).abs() <= e).all())
