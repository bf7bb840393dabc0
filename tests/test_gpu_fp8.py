"""The e4m3 products and their producers on the GPU against 64-bit forms (tests/fp8_plain.py). A product's tolerance is
the worst case of its f32 additions (gemm_bound) and the rounding to C's type; the producers' rows are the quantizer's exact
f32 result where the values it met are known, else e4m3 roundings of the 64-bit values."""
import numpy as np
import pytest
import torch

from tests import fp8_plain as P

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(qm, dev, N, K, M, seed, Ms=None):
    Ms = P.up(M, 16) if Ms is None else Ms
    Kp = P.up(K, 128)
    rng = np.random.default_rng(seed)
    w8 = P.random_e4m3((N, K), seed)
    wsc = torch.from_numpy(rng.uniform(0.5e-3, 2e-3, (P.up(N, 128) // 128, Kp // 128)).astype(np.float32))
    a8 = P.random_e4m3((Ms, Kp), seed + 1)
    a8[M:] = 0
    a8[:, K:] = 0
    asc = torch.from_numpy(rng.uniform(0.5e-2, 2e-2, (Kp // 128, Ms)).astype(np.float32))
    w = qm.Fp8Weight(w8.to(dev), wsc.to(dev))
    sums = P.gemm(*(t.to(dev) for t in (w8, wsc, a8, asc)), M)  # (in 64 bits there as well)
    return w, a8.view(torch.float8_e4m3fn).to(dev), asc.to(dev), [t.cpu() for t in sums]


def near(got, ref, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


SHAPES = [(1, 1, 1), (3, 40, 2), (64, 128, 1), (100, 128, 7), (128, 256, 16), (130, 300, 17), (257, 1000, 33), (512, 640, 64),
          (5184, 512, 65), (1000, 4096, 48), (640, 2048, 127), (384, 1024, 130), (2049, 896, 200), (256, 128, 500),
          (1153, 1536, 333), (512, 17408, 5), (448, 8200, 40), (2304, 2176, 260), (4096, 4096, 1), (768, 5120, 513)]


# every variant that the choice can make: few tokens by one or two fragments and 4, 8 or 16 waves; tiles of 4 to 8 token tiles, whole
# and in pieces, with one, two, three and no blocks left over of four, and more than 64 blocks
VARIANTS = [(256, 915, 18), (261, 2123, 17), (4184, 133, 17), (4157, 937, 17), (260, 129, 38), (260, 912, 35), (4202, 132, 33),
            (4207, 914, 33), (262, 934, 50), (4550, 940, 52), (8200, 2048, 16), (5000, 2100, 9), (258, 138, 1053), (266, 1679, 1143),
            (1845, 2456, 65), (901, 3983, 69), (272, 9425, 49), (461, 10184, 69), (3530, 1808, 68), (36725, 131, 65),
            (292, 2583, 2737), (8320, 2332, 68), (4200, 4041, 66), (35526, 130, 91), (33200, 141, 81), (262, 5405, 2699),
            (35154, 135, 97), (36787, 130, 113), (5000, 520, 4100), (16638, 8536, 342),
            (6440, 8581, 389), (4063, 9225, 324), (13391, 8435, 321), (14351, 8358, 524), (8420, 8327, 449), (1056, 8549, 2038)]


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("N,K,M", SHAPES + VARIANTS)
def test_product(qm, dev, N, K, M, out):
    w, a8, asc, (ref, *sums) = make(qm, dev, N, K, M, N + 3 * K + M)
    ws = qm.gemm_fp8_workspace(w, M)
    C = qm.gemm_fp8(w, a8, asc, M=M, out=out, ws=ws)
    kb = P.up(K, 128) // 128
    near(C, ref, P.gemm_bound(*sums, kb, out) + P.rounding(out, ref))
    # without the workspace: the same within the bound
    C = qm.gemm_fp8(w, a8, asc, M=M, out=F32)
    near(C, ref, P.gemm_bound(*sums, kb) + P.rounding(F32, ref))
    w.release()


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("N,K,M", [(130, 300, 3), (256, 512, 40), (576, 1024, 150), (640, 2048, 300)])
def test_accumulate_into_a_window(qm, dev, N, K, M, out):
    """accumulate 1 and 2 into columns of a wider C; what lies beside the window and behind the last token stays."""
    w, a8, asc, (ref, *sums) = make(qm, dev, N, K, M, N + M)
    bound = P.gemm_bound(*sums, P.up(K, 128) // 128, out)
    for ldc, off in ((N + 12, 4), (N + 7, 3)):
        g = torch.Generator().manual_seed(N)
        C0 = torch.randn((M + 2, ldc), generator=g).to(out)
        for acc in (0, 1, 2):
            C = C0.to(dev)
            qm.gemm_fp8(w, a8, asc, M=M, C=C, c_off=off, accumulate=acc, ws=qm.gemm_fp8_workspace(w, M))
            C, old = C.cpu(), C0.double()[:M, off:off + N]
            want = ref if acc == 0 else old + ref if acc == 1 else old * torch.sigmoid(old) * ref
            # (silu in f32: exp, a sum, a quotient, a product, each within two steps)
            extra = 0 if acc == 0 else P.U32 * want.abs() if acc == 1 else 12 * P.U32 * want.abs()
            b = bound if acc < 2 else bound * (old * torch.sigmoid(old)).abs() * 1.001
            near(C[:M, off:off + N], want, b + extra + P.rounding(out, want))
            C[:M, off:off + N] = C0[:M, off:off + N]
            assert torch.equal(C, C0)
    w.release()


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M", [1, 5, 40, 150, 300])
def test_nan_and_zero_rows_stay_their_own(qm, dev, M, out):
    """A token with a NaN has NaN results and no other token has; a weight row with a NaN likewise; a zero token gives zeros."""
    N, K = 320, 640
    w8 = P.random_e4m3((N, K), 5)
    a8 = P.random_e4m3((M, K), 6)
    a8[0, 130] = 0x7F
    w8[77, 300] = 0xFF
    if M > 2:
        a8[2] = 0
    w = qm.Fp8Weight(w8.to(dev), torch.ones((3, 5), device=dev))
    C = qm.gemm_fp8(w, a8.view(torch.float8_e4m3fn).to(dev), torch.ones((5, M), device=dev), out=out,
                    ws=qm.gemm_fp8_workspace(w, M)).float().cpu()
    nan = torch.zeros((M, N), dtype=torch.bool)
    nan[0], nan[:, 77] = True, True
    assert torch.equal(torch.isnan(C), nan)
    if M > 2:
        assert torch.equal(C[2][~nan[2]], torch.zeros(N - 1))
    w.release()


def test_weight_from_the_host_and_info(qm, dev):
    N, K, M = 200, 333, 4
    w8, a8 = P.random_e4m3((N, K), 1), P.random_e4m3((M, P.up(K, 128)), 2)
    a8[:, K:] = 0
    wsc = torch.rand((2, 3)) + 0.5
    a, s = a8.view(torch.float8_e4m3fn).to(dev), torch.ones((3, M), device=dev)
    here, there = qm.Fp8Weight(w8, wsc), qm.Fp8Weight(w8.view(torch.float8_e4m3fn).to(dev), wsc.to(dev))
    assert torch.equal(qm.gemm_fp8(here, a, s), qm.gemm_fp8(there, a, s))
    import ctypes
    r, k, kp = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    qm._call("qmatmul_fp8_info", here.handle, ctypes.byref(r), ctypes.byref(k), ctypes.byref(kp))
    assert (r.value, k.value, kp.value) == (N, K, 384) and here.nbytes >= 256 * 384 + 6 * 4
    # an unaligned source (rows of 333 bytes, base off by one)
    buf = torch.zeros(N * K + 1, dtype=torch.uint8, device=dev)
    buf[1:] = w8.to(dev).flatten()
    odd = qm.Fp8Weight(buf[1:].view(N, K), wsc.to(dev))
    assert torch.equal(qm.gemm_fp8(odd, a, s), qm.gemm_fp8(there, a, s))
    for w in (here, there, odd):
        w.release()


def test_rows_past_32_bit_offsets(qm, dev):
    """C rows further apart than 2^31 elements in all."""
    N, K, M = 96, 256, 4
    w, a8, asc, (ref, *sums) = make(qm, dev, N, K, M, 3)
    ld = 1 << 30
    C = torch.empty((M - 1) * ld + N, dtype=F16, device=dev).as_strided((M, N), (ld, 1))
    qm.gemm_fp8(w, a8, asc, M=M, C=C)
    near(C, ref, P.gemm_bound(*sums, 2, F16) + P.rounding(F16, ref))
    w.release()


@pytest.mark.parametrize("N,K,M", [(256, 1024, 3), (640, 2048, 40), (1024, 2048, 140), (512, 4096, 300)])
def test_graphs_and_streams(qm, dev, N, K, M):
    """Captured and replayed with eager work between; two streams at once with a workspace each; always the eager bits."""
    w, a8, asc, _ = make(qm, dev, N, K, M, M)
    want = qm.gemm_fp8(w, a8, asc, M=M, ws=qm.gemm_fp8_workspace(w, M))
    ws, C = qm.gemm_fp8_workspace(w, M), torch.empty((M, N), device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        qm.gemm_fp8(w, a8, asc, M=M, C=C, ws=ws)
    for _ in range(3):
        C.fill_(-1.0)
        graph.replay()
        assert torch.equal(qm.gemm_fp8(w, a8, asc, M=M, ws=qm.gemm_fp8_workspace(w, M)), want)
        torch.cuda.synchronize()
        assert torch.equal(C, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(qm.gemm_fp8(w, a8, asc, M=M, ws=qm.gemm_fp8_workspace(w, M)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    w.release()


def test_refusals(qm, dev):
    """What a product refuses once there is a weight: nothing is written, and the next call is unharmed."""
    N, K, M = 200, 300, 5
    w, a8, asc, (ref, *sums) = make(qm, dev, N, K, M, 1)
    C = torch.full((M, N), 7.0, device=dev)
    lib, st = qm.load_library(), qm._stream(None)
    call = lambda **k: lib.qmatmul_gemm_fp8(*{**dict(w=w.handle, a=a8.data_ptr(), s=asc.data_ptr(), M=M, Ms=16, C=C.data_ptr(), t=0,  # noqa: E731
                                                     ldc=N, off=0, acc=0, ws=None, wsb=0, st=st), **k}.values())
    assert call(M=0) == 0 and call(M=0, a=None, C=None) == 0
    for bad in (dict(a=None), dict(s=None), dict(C=None), dict(acc=3), dict(acc=-1), dict(a=a8.data_ptr() + 8), dict(s=asc.data_ptr() + 2),
                dict(C=C.data_ptr() + 2), dict(ws=C.data_ptr() + 16, wsb=1 << 20), dict(C=C.data_ptr() + 1, t=30)):
        assert call(**bad) == 1, bad
    for bad in (dict(M=-1), dict(M=17), dict(ldc=N - 1), dict(off=1), dict(off=-1), dict(off=2 ** 31 - 1, ldc=2 ** 31 - 1)):
        assert call(**bad) == 2, bad
    assert call(t=2) == 3 and call(t=14) == 3
    for bad in (lambda: qm.gemm_fp8(w, a8[:, :256].contiguous(), asc), lambda: qm.gemm_fp8(w, a8, asc[:, :8].contiguous()),
                lambda: qm.gemm_fp8(w, a8, asc.double()), lambda: qm.gemm_fp8(w, a8.float(), asc), lambda: qm.gemm_fp8(w, a8.cpu(), asc),
                lambda: qm.gemm_fp8(w, a8[::2], asc[:, ::2]), lambda: qm.gemm_fp8(w, a8, asc, out=torch.int32),
                lambda: qm.gemm_fp8(w, a8, asc, M=6, C=C), lambda: qm.gemm_fp8(w, a8, asc, M=M, C=C, out=BF16),
                lambda: qm.gemm_fp8(w, a8, asc, M=M, accumulate=1), lambda: qm.gemm_fp8(w, a8, asc, M=M, C=C, c_off=1),
                lambda: qm.gemm_fp8(w, a8, asc, M=M, C=C.t()), lambda: qm.gemm_fp8(w, a8, asc, M=17),
                lambda: qm.Fp8Weight(torch.zeros((4, 4), device=dev), torch.ones((1, 1), device=dev)),
                lambda: qm.Fp8Weight(torch.zeros((4, 200), dtype=torch.uint8, device=dev), torch.ones((1, 1), device=dev)),
                lambda: qm.Fp8Weight(torch.zeros((4, 4), dtype=torch.uint8, device=dev), torch.ones((1, 1))),
                lambda: qm.Fp8Weight(torch.zeros((4, 8), dtype=torch.uint8, device=dev)[:, ::2], torch.ones((1, 1), device=dev)),
                lambda: qm.quantize_fp8(torch.zeros((4, 4), dtype=torch.float64, device=dev)), lambda: qm.quantize_fp8(torch.zeros((4, 4))),
                lambda: qm.quantize_fp8(torch.zeros((4, 4), device=dev), M_stride=3), lambda: qm.quantize_fp8(torch.zeros((8, 4), device=dev).t()),
                lambda: qm.rmsnorm_fp8(torch.zeros((4, 4), device=dev), torch.ones(5, device=dev), 1e-6),
                lambda: qm.swiglu_fp8(torch.zeros((4, 7), device=dev), 4)):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert bool((C == 7.0).all())
    near(qm.gemm_fp8(w, a8, asc, M=M, C=C), ref, P.gemm_bound(*sums, 3) + P.rounding(F32, ref))
    w.release()
    with pytest.raises(qm.QMatmulError):
        qm.gemm_fp8(w, a8, asc, M=M, C=C)


def test_activations_of_other_bytes(qm, dev):
    """Bytes of e4m3 are taken as such; other types of one byte are not read as e4m3."""
    w, a8, asc, _ = make(qm, dev, 96, 256, 3, 1)
    want = qm.gemm_fp8(w, a8, asc)
    assert torch.equal(qm.gemm_fp8(w, a8.view(torch.uint8), asc), want)
    for t in (torch.int8, torch.float8_e5m2, torch.float8_e4m3fnuz, torch.bool):
        with pytest.raises(qm.QMatmulError):
            qm.gemm_fp8(w, a8.view(t), asc)


def test_columns_beside_a_view_are_no_room(qm, dev):
    """C as a view of some columns: rows that end past its last column are refused, also where the matrix behind has the room."""
    N, K, M = 200, 300, 5
    w, a8, asc, (ref, *sums) = make(qm, dev, N, K, M, 1)
    buf = torch.full((M + 3, 2 * N), 7.0, device=dev)
    for C, k in ((buf[:, :N], dict(c_off=1)), (buf[:, :N - 1], {}), (buf[:, N // 2:N + N // 2], dict(c_off=N // 2)), (buf[:M - 1, :N], {})):
        with pytest.raises(qm.QMatmulError):
            qm.gemm_fp8(w, a8, asc, M=M, C=C, **k)
    assert bool((buf == 7.0).all())
    qm.gemm_fp8(w, a8, asc, M=M, C=buf[:, 50:50 + N])
    near(buf[:M, 50:50 + N], ref, P.gemm_bound(*sums, 3) + P.rounding(F32, ref))
    assert bool((buf[M:] == 7.0).all()) and bool((buf[:, :50] == 7.0).all()) and bool((buf[:, 50 + N:] == 7.0).all())


@pytest.mark.parametrize("N,K", [(512, 17408), (5184, 5120), (17408, 5120)])
def test_workspaces_are_bounded_and_optional(qm, dev, N, K):
    """Never more than 64 MiB; a larger or smaller one than asked for gives the bound's result too."""
    wsc = torch.rand((P.up(N, 128) // 128, K // 128), device=dev) * 1e-3
    w = qm.Fp8Weight(P.random_e4m3((N, K), 3).to(dev), wsc)
    sizes = [qm.load_library().qmatmul_gemm_fp8_workspace_size(w.handle, M) for M in list(range(1, 200, 7)) + [333, 777, 4096, 100000]]
    assert max(sizes) <= 64 << 20 and sizes[0] == 0 and any(sizes)
    M = 70
    a8 = P.random_e4m3((M, K), 4).to(dev).view(torch.float8_e4m3fn)
    asc = torch.rand((K // 128, M), device=dev) * 1e-2
    w8 = P.random_e4m3((N, K), 3).to(dev)
    A = P.gemm(w8, wsc, a8, asc, M)[1]
    need = qm.load_library().qmatmul_gemm_fp8_workspace_size(w.handle, M)
    whole = qm.gemm_fp8(w, a8, asc)
    for n in (need, 64 << 20, max(256, need - 256)):
        C = qm.gemm_fp8(w, a8, asc, ws=torch.empty(n, dtype=torch.uint8, device=dev))
        off = (C.double() - whole.double()).abs()  # (both are within the worst case of f32 sums of the absolute values)
        assert bool((off <= 2 * P.gemm_bound(A, 0, K // 128)).all())
    w.release()


# ---- producers -------------------------------------------------------------------------------------------------------
def same(a8, asc, q, sc, M):
    assert torch.equal(P.value(a8.cpu())[:M], q), "e4m3 rows"
    assert torch.equal(asc.cpu()[:, :M], sc), "scales"
    assert not a8.cpu().view(torch.uint8)[M:].any() and not asc.cpu()[:, M:].any(), "padding"


ROWS = [(1, 16, 5120), (7, 8, 2048), (3, 3, 17408), (2, 4, 96), (5, 5, 1), (4, 16, 1001), (300, 304, 640), (33, 48, 2050)]


@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("M,Ms,K", ROWS)
def test_quantize(qm, dev, M, Ms, K, x_type):
    rng = np.random.default_rng(M + K)
    x = torch.from_numpy((rng.standard_normal((M, K)) * 10.0 ** rng.uniform(-3, 3, (M, K))).astype(np.float32))
    x[0, :128] = 0.0
    x = x.to(x_type)
    q, sc = P.quantize32(x.float().numpy())
    same(*qm.quantize_fp8(x.to(dev), M_stride=Ms), q, sc, M)
    wide = torch.full((M, K + 9), 7.0, dtype=x_type, device=dev)  # rows of another stride and alignment
    wide[:, 5:5 + K] = x.to(dev)
    same(*qm.quantize_fp8(wide[:, 5:5 + K], M_stride=Ms), q, sc, M)


def test_quantize_extremes(qm, dev):
    """Blocks of the largest, tiny, zero, infinite and NaN values: no other block or row is touched."""
    x = torch.ones((6, 384))
    x[0, :128] = 3.0e38
    x[1, :128] = 2.0 ** -101
    x[2, :128] = 2.0 ** -100
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    x[5, :128] = -0.0
    a8, asc = qm.quantize_fp8(x.to(dev))
    v, s = P.value(a8.cpu()), asc.cpu()
    ones = torch.full((128,), 448.0, dtype=torch.float64)
    assert torch.equal(v[0, :128], ones) and s[0, 0] == np.float32(3.0e38) / np.float32(448)
    assert not v[1, :128].any() and s[0, 1] == 0 and torch.equal(v[2, :128], ones) and s[0, 2] == np.float32(2.0 ** -100 / 448)
    assert torch.isinf(s[0, 3]) and torch.isnan(v[3, 5]) and not v[3, :5].any()
    assert torch.isnan(v[4, 7]) and torch.isnan(v[4]).sum() == 1 and s[0, 4] == np.float32(1 / 448)
    assert not v[5, :128].any() and s[0, 5] == 0
    assert torch.equal(v[:, 128:], torch.full((6, 256), 448.0, dtype=torch.float64)) and bool((s[1:] == np.float32(1 / 448)).all())
    w = qm.Fp8Weight(torch.full((16, 384), 0x38, dtype=torch.uint8, device=dev), torch.ones((1, 3), device=dev))  # ones
    C = qm.gemm_fp8(w, a8, asc).cpu()
    assert torch.isnan(C[3]).all() and torch.isnan(C[4]).all() and torch.isfinite(C[[1, 2, 5]]).all()
    w.release()


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("M,Ms,K", ROWS + [(2, 2, 40000), (260, 260, 20000)])
def test_rmsnorm(qm, dev, M, Ms, K, x_type):
    rng = np.random.default_rng(M + K)
    x = torch.from_numpy((rng.standard_normal((M, K)) * rng.uniform(0.1, 10)).astype(np.float32)).to(x_type)
    w = torch.from_numpy(rng.uniform(0.2, 2.0, K).astype(np.float32))
    a8, asc, h = qm.rmsnorm_fp8(x.to(dev), w.to(dev), 1e-6, M_stride=Ms, want_h=True)
    x64 = x.double()
    y = x64 / torch.sqrt((x64 * x64).mean(1, keepdim=True) + 1e-6) * w.double()
    e = P.norm_error(K, 8 * ((K + 2047) // 2048))
    near(h, y, e * y.abs() + 1e-40)
    q, sc = P.quantize32(h.cpu().numpy())  # the quantizer's exact result on the kernel's own y
    same(a8, asc, q, sc, M)
    b8, bsc, none = qm.rmsnorm_fp8(x.to(dev), w.to(dev), 1e-6, M_stride=Ms)
    assert none is None and torch.equal(b8.view(torch.uint8), a8.view(torch.uint8)) and torch.equal(bsc, asc)


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("x_type", [F32, F16, BF16])
@pytest.mark.parametrize("M,Ms,F", [(1, 16, 17408), (5, 8, 512), (2, 2, 97), (260, 260, 1024), (19, 32, 2184)])
def test_swiglu(qm, dev, gelu, M, Ms, F, x_type):
    rng = np.random.default_rng(F + M)
    gu = torch.from_numpy((rng.standard_normal((M, 2 * F)) * 3).astype(np.float32)).to(x_type)
    a8, asc = qm.swiglu_fp8(gu.to(dev), F, gelu=gelu, M_stride=Ms)
    g, u = gu.double()[:, :F], gu.double()[:, F:]
    z = 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3) if gelu else g
    y = g * torch.sigmoid(z) * u
    # silu: exp (two steps), a sum, a quotient, a product; gelu: tanh's argument (|z| U32 times its slope, below 4 in all), tanh, then
    # 1 + tanh, which cancels where g < 0: absolute against |g u|
    err = (32 * P.U32 * (g * u).abs()) if gelu else 8 * P.U32 * y.abs()
    p = torch.zeros((2, M, P.up(F, 128)), dtype=torch.float64)
    p[0, :, :F], p[1, :, :F] = y, err
    top, terr = (v.view(M, -1, 128) for v in p)
    top, terr = top.abs().amax(2), terr.amax(2)
    assert bool(((asc.cpu().double()[:, :M].T - top / 448).abs() <= terr / 448 + 2 * P.U32 * top / 448).all())
    s = (448 / top)[:, :, None].expand(-1, -1, 128).reshape(M, -1)
    v = p[0] * s
    e = (p[1] * s) + v.abs() * ((terr / top)[:, :, None].expand(-1, -1, 128).reshape(M, -1) + 4 * P.U32)
    # (an error near a border is a whole step there: the border itself lies half a step from both)
    assert P.near_e4m3(P.value(a8.cpu())[:M], v, 1.1 * e)
    assert not a8.cpu().view(torch.uint8)[M:].any() and not a8.cpu().view(torch.uint8)[:, F:].any()


@pytest.mark.parametrize("gelu", [False, True])
def test_swiglu_extremes(qm, dev, gelu):
    """Gates far out of the exponential's range: the gate itself, or nothing; an infinity or a NaN stays in its row."""
    gu = torch.ones((5, 512))
    gu[0, :4] = torch.tensor([1e30, -1e30, 90.0, -90.0])
    gu[1, 0], gu[2, 0], gu[3, 0], gu[4, 256] = float("inf"), float("-inf"), float("nan"), float("nan")
    a8, asc = qm.swiglu_fp8(gu.to(dev), 256, gelu=gelu)
    v, s = P.value(a8.cpu()), asc.cpu().double()
    assert v[0, 0] == 448 and abs(s[0, 0] * 448 / 1e30 - 1) < 1e-6 and not v[0, 1:128].any()
    assert torch.isfinite(v[:, 128:]).all() and torch.isfinite(s[1]).all()
    ones = qm.Fp8Weight(torch.full((16, 256), 0x38, dtype=torch.uint8, device=dev), torch.ones((1, 2), device=dev))
    C = qm.gemm_fp8(ones, a8, asc).cpu()
    assert torch.isfinite(C[0]).all() and not torch.isfinite(C[1]).any() and torch.isnan(C[3]).all() and torch.isnan(C[4]).all()
    gu = torch.full((1, 256), 90.0)  # (a block of far gates alone: what is left of -90 is below 2^-100)
    gu[0, 64:128] = -90.0
    a8, asc = qm.swiglu_fp8(gu.to(dev), 128, gelu=gelu)
    v = P.value(a8.cpu())
    assert bool((v[0, :64] == 448).all()) and not v[0, 64:].any()
    ones.release()


def test_ffn_run(qm, dev):
    """Norm, gate and up, gating, down, as an FFN layer uses them, with C in bf16 and f32; each product against 64 bits on the
    activations that it met."""
    E, Fw = 640, 1152
    ws = {n: (P.random_e4m3(s, i), torch.rand((P.up(s[0], 128) // 128, P.up(s[1], 128) // 128)) * 1e-3 + 1e-4)
          for i, (n, s) in enumerate((("gate", (Fw, E)), ("up", (Fw, E)), ("down", (E, Fw))))}
    h = {n: qm.Fp8Weight(a.to(dev), b.to(dev)) for n, (a, b) in ws.items()}
    for M in (1, 21, 150):
        x = torch.randn((M, E), generator=torch.Generator().manual_seed(M)).to(dev)
        norm = torch.rand(E, device=dev) + 0.5
        a8, asc, _ = qm.rmsnorm_fp8(x, norm, 1e-6, M_stride=P.up(M, 16))
        gu = torch.empty((M, 2 * Fw), dtype=BF16, device=dev)
        for n, off in (("gate", 0), ("up", Fw)):
            qm.gemm_fp8(h[n], a8, asc, M=M, C=gu, c_off=off, ws=qm.gemm_fp8_workspace(h[n], M))
            ref, *sums = P.gemm(*ws[n], a8.cpu(), asc.cpu(), M)
            near(gu[:, off:off + Fw], ref, P.gemm_bound(*sums, E // 128, BF16) + P.rounding(BF16, ref))
        b8, bsc = qm.swiglu_fp8(gu, Fw, M_stride=P.up(M, 16))
        y = x.clone()
        qm.gemm_fp8(h["down"], b8, bsc, M=M, C=y, accumulate=1, ws=qm.gemm_fp8_workspace(h["down"], M))
        ref, *sums = P.gemm(*ws["down"], b8.cpu(), bsc.cpu(), M)
        ref = ref + x.double().cpu()
        near(y, ref, P.gemm_bound(*sums, Fw // 128) + 2 * P.rounding(F32, ref))
    for w in h.values():
        w.release()
