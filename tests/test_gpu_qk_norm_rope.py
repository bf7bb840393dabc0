"""The q/k head norm + rotation on the GPU against its 64-bit form (tests/fp8_plain.py)."""
import numpy as np
import pytest
import torch

from tests import fp8_plain as P

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def inv_freq(rot, theta=1e6):
    i = np.arange(rot // 2, dtype=np.float64)
    return torch.from_numpy((theta ** (-2.0 * i / max(1, rot))).astype(np.float32))


def positions(T, axes, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 300000, (axes, T), generator=g, dtype=torch.int32)
    p[:, :1] = 0
    p[0, -1] = 2 ** 31 - 1 if T > 2 else 5
    return p


def check(got, x, w, eps, pos, f, sections, turns, adjacent, scale, out, seq):
    y, B = P.rotated(x.double(), None if w is None else w.double(), eps, pos, f, sections, turns, adjacent, scale)
    # norm; cosine and sine: turns reduced in f64 to 2^-22 of a radian at the last position (2^31 / 2 pi turns, 2^-53 each way), rounded
    # to f32 (pi U32 at half a turn), two steps of their own, the scale; two products and a sum
    e = (P.norm_error(x.shape[2], seq) if w is not None else 0) + (4 + np.pi + 2 + 1 + 3) * P.U32
    bound = e * B + P.rounding(out, y) + 1e-40
    off = (got.double().cpu() - y).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


CASES = [  # T, HQ, HK, D, rot
    (1, 1, 1, 2, 2), (1, 24, 4, 256, 64), (3, 8, 2, 128, 128), (5, 3, 1, 80, 80), (7, 4, 4, 64, 32), (2, 2, 1, 512, 512),
    (4, 5, 5, 96, 48), (9, 2, 1, 130, 50), (33, 6, 3, 40, 10), (130, 16, 8, 128, 64), (2, 3, 2, 510, 254), (6, 4, 2, 128, 0),
    (1100, 4, 2, 64, 64), (1027, 3, 1, 192, 96), (17, 0, 3, 64, 64), (17, 3, 0, 64, 64),
]


@pytest.mark.parametrize("xt,out", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("T,HQ,HK,D,rot", CASES)
def test_one_axis(qm, dev, T, HQ, HK, D, rot, xt, out):
    g = torch.Generator().manual_seed(T + D)
    x = (torch.randn((T, (HQ + 2 * HK) * D), generator=g) * 3).to(xt)
    wq, wk = torch.rand(D, generator=g) + 0.5, torch.rand(D, generator=g) + 0.5
    pos, f = positions(T, 1, D)[0], inv_freq(rot)
    for adjacent in (False, True):
        for norm in (True, False):
            q, k = qm.qk_norm_rope(x.to(dev), HQ, HK, D, pos.to(dev), f.to(dev), wq=wq.to(dev) if norm else None,
                                   wk=wk.to(dev) if norm else None, adjacent=adjacent, out=out)
            assert q.shape == (T, HQ, D) and k.shape == (T, HK, D) and q.dtype == out
            for got, a, H, w in ((q, 0, HQ, wq), (k, HQ * D, HK, wk)):
                check(got, x[:, a:a + H * D].reshape(T, H, D), w if norm else None, 1e-6, pos[None], f, [rot // 2], False,
                      adjacent, 1.0, out, 8)


@pytest.mark.parametrize("turns", [False, True])
@pytest.mark.parametrize("T,HQ,HK,D,rot,sections", [
    (5, 4, 2, 128, 128, (16, 24, 24)), (777, 6, 1, 256, 64, (11, 11, 10)), (31, 4, 4, 80, 80, (20, 20)),
    (3, 2, 1, 96, 96, (12, 12, 12, 12)), (4, 2, 2, 64, 64, (32, 0, 0)), (4, 2, 2, 64, 64, (0, 16, 16)), (6, 1, 1, 30, 22, (5, 3, 3))])
def test_several_axes(qm, dev, T, HQ, HK, D, rot, sections, turns):
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, (HQ + HK) * D), generator=g)
    wq = torch.rand(D, generator=g) + 0.5
    pos, f = positions(T, len(sections), T), inv_freq(rot)
    pos[-1] *= -1  # (a position may be negative)
    q, k = qm.qk_norm_rope(x.to(dev), HQ, HK, D, pos.to(dev), f.to(dev), wq=wq.to(dev), sections=sections, turns=turns, scale=1.25)
    check(q, x[:, :HQ * D].reshape(T, HQ, D), wq, 1e-6, pos, f, sections, turns, False, 1.25, F32, 8)
    check(k, x[:, HQ * D:].reshape(T, HK, D), None, 1e-6, pos, f, sections, turns, False, 1.25, F32, 8)


def test_one_axis_of_several_is_one_axis(qm, dev):
    """Equal positions on every axis turn as one axis does, bit for bit, in either order."""
    T, D = 40, 128
    x = torch.randn((T, 6 * D), device=dev)
    f, p = inv_freq(D).to(dev), torch.arange(T, dtype=torch.int32, device=dev)
    want = qm.qk_norm_rope(x, 4, 2, D, p, f)
    for turns in (False, True):
        got = qm.qk_norm_rope(x, 4, 2, D, p.expand(3, T).contiguous(), f, sections=(24, 20, 20), turns=turns)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("xt", [F32, BF16])
def test_strides_and_in_place(qm, dev, xt):
    """Heads apart from each other (a gate between the query heads), rows of a wider matrix, unaligned columns, outputs in
    one buffer, and in place: the same bits, nothing else written."""
    T, HQ, HK, D = 21, 4, 2, 128
    g = torch.Generator().manual_seed(1)
    heads = torch.randn((T, HQ + HK, D), generator=g).to(xt).to(dev)
    w = (torch.rand(D, generator=g) + 0.5).to(dev)
    f, p = inv_freq(64).to(dev), torch.arange(7, 7 + T, dtype=torch.int32, device=dev)
    kw = dict(wq=w, wk=w)
    want = qm.qk_norm_rope(heads.view(T, -1), HQ, HK, D, p, f, **kw)
    # query heads 2 D apart, key heads D + 4 apart
    x = torch.full((T, 3000), 9.0, dtype=xt, device=dev)
    x[:, 8:8 + 2 * HQ * D].view(T, HQ, 2 * D)[:, :, :D] = heads[:, :HQ]
    k_off = 8 + 2 * HQ * D
    for h in range(HK):
        x[:, k_off + h * (D + 4):k_off + h * (D + 4) + D] = heads[:, HQ + h]
    got = qm.qk_norm_rope(x, HQ, HK, D, p, f, q_off=8, q_hs=2 * D, k_off=k_off, k_hs=D + 4, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # unaligned columns: by the element (another order of the squares' sum)
    y = torch.zeros((T, (HQ + HK) * D + 5), dtype=xt, device=dev)
    y[:, 3:3 + (HQ + HK) * D] = heads.view(T, -1)
    q, k = qm.qk_norm_rope(y, HQ, HK, D, p, f, q_off=3, **kw)
    for a, b in ((q, want[0]), (k, want[1])):
        assert float((a.double() - b.double()).abs().max()) <= (2.0 ** -7 if xt == BF16 else 2.0 ** -19) * float(b.abs().max())
    # both outputs in one buffer of rows
    buf = torch.full((T + 1, (HQ + HK) * D + 16), -3.0, dtype=xt, device=dev)
    qm.qk_norm_rope(heads.view(T, -1), HQ, HK, D, p, f, q=buf[:T, 8:8 + HQ * D], k=buf[:T, 8 + HQ * D:8 + (HQ + HK) * D], **kw)
    assert torch.equal(buf[:T, 8:8 + HQ * D].reshape(T, HQ, D), want[0])
    assert torch.equal(buf[:T, 8 + HQ * D:-8].reshape(T, HK, D), want[1])
    assert bool((buf[T] == -3).all()) and bool((buf[:, :8] == -3).all()) and bool((buf[:, -8:] == -3).all())
    # in place
    z = heads.clone().view(T, -1)
    qm.qk_norm_rope(z, HQ, HK, D, p, f, q=z[:, :HQ * D], k=z[:, HQ * D:], **kw)
    assert torch.equal(z[:, :HQ * D].reshape(T, HQ, D), want[0]) and torch.equal(z[:, HQ * D:].reshape(T, HK, D), want[1])


def test_one_token_in_place(qm, dev):
    """A single row, its heads rotated where they lie, whatever row stride the views of it carry."""
    HQ, HK, D = 4, 2, 64
    x = torch.randn((1, (HQ + HK) * D), generator=torch.Generator().manual_seed(3)).to(dev)
    f, p, w = inv_freq(D).to(dev), torch.tensor([11], dtype=torch.int32, device=dev), torch.ones(D, device=dev)
    want = qm.qk_norm_rope(x, HQ, HK, D, p, f, wq=w)
    n = HQ * D
    for q_of, k_of in ((lambda z: z[:, :n], lambda z: z[:, n:]), (lambda z: z[0, :n].view(1, HQ, D), lambda z: z[0, n:].view(1, HK, D)),
                       (lambda z: z[0, :n].view(1, n), lambda z: z[0, n:].view(1, HK * D))):
        z = x.clone()
        qm.qk_norm_rope(z, HQ, HK, D, p, f, wq=w, q=q_of(z), k=k_of(z))
        assert torch.equal(z[:, :n].view(1, HQ, D), want[0]) and torch.equal(z[:, n:].view(1, HK, D), want[1])


def test_infinities_and_nan_stay_in_their_head(qm, dev):
    T, D = 3, 64
    x = torch.randn((T, 4 * D), generator=torch.Generator().manual_seed(0))
    f, p = inv_freq(D).to(dev), torch.arange(T, dtype=torch.int32, device=dev)
    w = torch.ones(D, device=dev)
    want = qm.qk_norm_rope(x.to(dev), 2, 2, D, p, f, wq=w, wk=w)
    x[1, D + 3], x[2, 2 * D] = float("nan"), float("inf")
    got = qm.qk_norm_rope(x.to(dev), 2, 2, D, p, f, wq=w, wk=w)
    assert torch.isnan(got[0][1, 1]).all() and torch.isnan(got[1][2, 0]).any()
    keep_q, keep_k = torch.ones((T, 2), dtype=torch.bool), torch.ones((T, 2), dtype=torch.bool)
    keep_q[1, 1], keep_k[2, 0] = False, False
    assert torch.equal(got[0].cpu()[keep_q], want[0].cpu()[keep_q]) and torch.equal(got[1].cpu()[keep_k], want[1].cpu()[keep_k])


def test_zero_rows_and_no_tokens(qm, dev):
    f = inv_freq(64).to(dev)
    q, k = qm.qk_norm_rope(torch.zeros((2, 192), device=dev), 2, 1, 64, torch.zeros(2, dtype=torch.int32, device=dev), f,
                           wq=torch.ones(64, device=dev))
    assert not q.any() and not k.any()
    q, k = qm.qk_norm_rope(torch.zeros((0, 192), device=dev), 2, 1, 64, torch.zeros(0, dtype=torch.int32, device=dev), f)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)


def test_rows_past_32_bit_offsets(qm, dev):
    T, D, ld = 4, 64, 1 << 30
    x = torch.empty((T - 1) * ld + 2 * D, dtype=BF16, device=dev).as_strided((T, 2 * D), (ld, 1))
    x.copy_(torch.randn((T, 2 * D), generator=torch.Generator().manual_seed(0)))
    f, p = inv_freq(D).to(dev), torch.arange(T, dtype=torch.int32, device=dev)
    want = qm.qk_norm_rope(x.contiguous(), 1, 1, D, p, f)
    got = qm.qk_norm_rope(x, 1, 1, D, p, f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    qm.qk_norm_rope(x, 1, 1, D, p, f, q=x[:, :D], k=x[:, D:])
    assert torch.equal(x[:, :D].contiguous().view(T, 1, D), want[0]) and torch.equal(x[:, D:].contiguous().view(T, 1, D), want[1])


def test_graph_and_streams(qm, dev):
    T, HQ, HK, D = 50, 8, 2, 128
    x = torch.randn((T, (HQ + HK) * D), device=dev)
    w = torch.rand(D, device=dev) + 0.5
    f, p = inv_freq(D).to(dev), torch.arange(T, dtype=torch.int32, device=dev)
    want = qm.qk_norm_rope(x, HQ, HK, D, p, f, wq=w, wk=w)
    q, k = torch.empty_like(want[0]), torch.empty_like(want[1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        qm.qk_norm_rope(x, HQ, HK, D, p, f, wq=w, wk=w, q=q, k=k)
    for step in range(3):
        p.add_(1)  # the next position: read at the replay
        graph.replay()
        now = qm.qk_norm_rope(x, HQ, HK, D, p, f, wq=w, wk=w)
        torch.cuda.synchronize()
        assert torch.equal(q, now[0]) and torch.equal(k, now[1]) and not torch.equal(q, want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = qm.qk_norm_rope(x, HQ, HK, D, p, f, wq=w, wk=w)
    s.synchronize()
    assert torch.equal(got[0], q) and torch.equal(got[1], k)


def test_refusals(qm, dev):
    T, D = 4, 64
    x, f = torch.zeros((T, 6 * D), device=dev), inv_freq(D).to(dev)
    p = torch.arange(T, dtype=torch.int32, device=dev)
    ok = lambda **k: qm.qk_norm_rope(*{**dict(x=x, HQ=4, HK=2, D=D, pos=p, f=f), **{n: k.pop(n) for n in ("x", "pos", "f", "D", "HQ") if n in k}}.values(), **k)  # noqa: E731
    ok()
    for bad in (dict(pos=p.long()), dict(pos=p[:3]), dict(pos=p.cpu()), dict(f=f.double()), dict(f=inv_freq(2 * D + 2).to(dev)), dict(D=63),
                dict(HQ=5), dict(x=x.double()), dict(x=x.cpu()), dict(x=x.t()), dict(wq=torch.ones(D - 1, device=dev)),
                dict(wk=torch.ones(D, device=dev).half()), dict(sections=(16, 15)), dict(sections=(32, 0)), dict(pos=p.expand(3, T), sections=(12, 10, 10)),
                dict(pos=p.expand(5, T).contiguous(), sections=(8, 8, 8, 4, 4)), dict(q=torch.zeros((T, 3 * D), device=dev)),
                dict(q=x[:, D:5 * D]), dict(k=x[:, 4 * D:].to(torch.bfloat16), out=F32), dict(out=torch.int8), dict(q_off=3 * D), dict(k_hs=D - 2),
                dict(q=torch.zeros((T, D, 4), device=dev).transpose(1, 2))):
        with pytest.raises(qm.QMatmulError):
            ok(**bad)


@pytest.mark.parametrize("M", [1, 5, 70, 200])
def test_attention_input_run(qm, dev, M):
    """The input side of an attention layer: norm -> e4m3 rows -> QKV product -> head norms and rotation, in place on the
    product's rows; the last step against 64 bits on the rows that it met, and the whole against each step alone."""
    E, HQ, HK, D = 640, 4, 2, 128
    N = (HQ + 2 * HK) * D
    w8, wsc = P.random_e4m3((N, E), M), torch.rand((N // 128, E // 128)) * 1e-3 + 1e-4
    w = qm.Fp8Weight(w8.to(dev), wsc.to(dev))
    g = torch.Generator().manual_seed(M)
    x = torch.randn((M, E), generator=g).to(dev)
    norm, wq, wk = (torch.rand(n, generator=g).to(dev) + 0.5 for n in (E, D, D))
    f, p = inv_freq(64), torch.arange(M, dtype=torch.int32)
    a8, asc, _ = qm.rmsnorm_fp8(x, norm, 1e-6, M_stride=P.up(M, 16))
    qkv = qm.gemm_fp8(w, a8, asc, M=M, out=BF16, ws=qm.gemm_fp8_workspace(w, M))
    ref, *sums = P.gemm(w8, wsc, a8.cpu(), asc.cpu(), M)
    assert bool(((qkv.double().cpu() - ref).abs() <= P.gemm_bound(*sums, E // 128, BF16) + P.rounding(BF16, ref)).all())
    rows = qkv.cpu()
    q, k = qm.qk_norm_rope(qkv, HQ, HK, D, p.to(dev), f.to(dev), wq=wq, wk=wk, q=qkv[:, :HQ * D], k=qkv[:, HQ * D:(HQ + HK) * D])
    check(q.reshape(M, HQ, D), rows[:, :HQ * D].reshape(M, HQ, D), wq.cpu(), 1e-6, p[None], f, [32], False, False, 1.0, BF16, 8)
    check(k.reshape(M, HK, D), rows[:, HQ * D:(HQ + HK) * D].reshape(M, HK, D), wk.cpu(), 1e-6, p[None], f, [32], False, False, 1.0, BF16, 8)
    assert torch.equal(qkv[:, (HQ + HK) * D:].cpu(), rows[:, (HQ + HK) * D:])  # (the values stay)
    w.release()
