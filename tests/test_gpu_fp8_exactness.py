"""How exact the e4m3 products are as a whole (the bound of each single result, in test_gpu_fp8, is that of its worst case, which a
long row never comes near): the error before C's rounding, and the norm of all errors."""
import pytest
import torch

from tests import fp8_plain as P
from tests import test_gpu_fp8 as G

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rms(x):
    return float(x.double().pow(2).mean().sqrt())


def dropped(a, w):
    """What the fp8 matrix pipe may leave out of the products of e4m3 values a [M, K], w [N, K], as one standard deviation [M, N]:
    of each eight, a product's part below 2^-13 of the largest product (none where it ends above that), their signs
    independent."""
    total = torch.zeros((len(a), len(w)), dtype=torch.float64, device=a.device)
    for k in range(0, a.shape[1], 8):
        p = a[:, None, k:k + 8] * w[None, :, k:k + 8]
        top = p.abs().amax(2, keepdim=True)
        unit = 2.0 ** -13 * torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -100))))
        whole = torch.trunc(p / unit) * unit == p
        loss = torch.where(whole, 0.0, torch.minimum(p.abs(), 2.0 ** -13 * top))
        total += loss.pow(2).sum(2)
    return total.sqrt()


def quantized(n, K, seed):
    """e4m3 bytes of normal values, each 128 of them scaled to the largest."""
    x = torch.randn((n, K), generator=torch.Generator().manual_seed(seed)).view(n, -1, 128)
    return (x * (448.0 / x.abs().amax(2, keepdim=True))).view(n, K).to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("kind", ["normal", "codes"])
@pytest.mark.parametrize("N,K,M", [(96, 1024, 5), (128, 2048, 16), (96, 1024, 40), (160, 1024, 150), (128, 4096, 140)])
def test_error_before_the_rounding(qm, dev, N, K, M, kind):
    """A C of 16 bits that holds the negated result, rounded, and the product added: what remains is 2^-11 of the result, so its rounding
    hides nothing. The fp8 pipe drops no more than `dropped`; f32 additions lose a step (2 U32) each, as a random walk of 132 + K / 128."""
    w8, a8 = (quantized(N, K, 1), quantized(M, K, 2)) if kind == "normal" else (P.random_e4m3((N, K), 1), P.random_e4m3((M, K), 2))
    w8, a8 = w8.to(dev), a8.to(dev)
    wsc, asc = (torch.full(s, v, device=dev) for s, v in (((P.up(N, 128) // 128, K // 128), 2.0 ** -8), ((K // 128, M), 2.0 ** -9)))
    w, scale = qm.Fp8Weight(w8, wsc), 2.0 ** -17
    ref = P.gemm(w8, wsc, a8, asc, M)[0]
    bound = rms(dropped(P.value(a8), P.value(w8)) * scale)
    walk = 2 * P.U32 * (132 + K // 128) ** 0.5 * rms(ref)
    for ws in (qm.gemm_fp8_workspace(w, M), None):
        C = -ref.to(F16)
        left = ref + C.double()  # (exact: what the kernel's sum plus C would be)
        qm.gemm_fp8(w, a8, asc, M=M, C=C, accumulate=1, ws=ws)
        err = rms(C.double() - left)
        print(f"{kind} {N} x {K}, {M}: {err / rms(ref):.2e} of the result, bound {bound / rms(ref):.2e}")
        assert err <= bound + walk + 2.0 ** -11 * rms(left)
        err = rms(qm.gemm_fp8(w, a8, asc, M=M, ws=ws).double() - ref)
        assert err <= walk + P.U32 * rms(ref)
    w.release()


@pytest.mark.parametrize("out", [BF16, F16])
@pytest.mark.parametrize("N,K,M", G.SHAPES + G.VARIANTS)
def test_norm_of_all_errors(qm, dev, N, K, M, out):
    """The rounding's norm (of the exact results: where there are a thousand, within a tenth; else the largest it can be) and the pipe's
    loss, at most 2^-13 sqrt(8) of the result: eight products of independent signs, each short of 2^-13 of the largest."""
    w, a8, asc, (ref, *_) = G.make(qm, dev, N, K, M, N + 3 * K + M)
    C = qm.gemm_fp8(w, a8, asc, M=M, out=out, ws=qm.gemm_fp8_workspace(w, M)).double().cpu()
    rounding = 1.1 * rms(ref.to(out).double() - ref) if N * M >= 1000 else P.HALF[out] * rms(ref)
    assert rms(C - ref) <= rounding + 2.0 ** -13 * 8 ** 0.5 * rms(ref)
    w.release()
