"""A batch of no tokens through producers, products and rotation: empty results, or (padded) rows of zeros."""
import pytest
import torch

from tests import fp8_plain as P

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("Ms", [None, 0, 1, 16])
def test_a_layer_of_no_tokens(qm, dev, x_type, Ms):
    E, Fw = 640, 1152
    w = [qm.Fp8Weight(P.random_e4m3(s, 1).to(dev), torch.ones((P.up(s[0], 128) // 128, P.up(s[1], 128) // 128), device=dev))
         for s in ((2 * Fw, E), (E, Fw))]
    x = torch.empty((0, E), dtype=x_type, device=dev)
    rows = Ms or 0

    def zeros(a8, asc, K):
        assert a8.shape == (rows, P.up(K, 128)) and asc.shape == (P.up(K, 128) // 128, rows)
        assert a8.dtype == torch.float8_e4m3fn and not a8.view(torch.uint8).any() and not asc.any()
    a8, asc = qm.quantize_fp8(x, M_stride=Ms)
    zeros(a8, asc, E)
    a8, asc, h = qm.rmsnorm_fp8(x, torch.ones(E, device=dev), 1e-6, M_stride=Ms, want_h=True)
    zeros(a8, asc, E)
    assert h.shape == (0, E)
    gu = qm.gemm_fp8(w[0], a8, asc, M=0, out=x_type, ws=qm.gemm_fp8_workspace(w[0], 0))
    assert gu.shape == (0, 2 * Fw) and gu.dtype == x_type
    a8, asc = qm.swiglu_fp8(gu, Fw, M_stride=Ms)
    zeros(a8, asc, Fw)
    assert qm.gemm_fp8(w[1], a8, asc, M=0).shape == (0, E)
    q, k = qm.qk_norm_rope(gu, 2, 1, 64, torch.empty(0, dtype=torch.int32, device=dev), torch.ones(32, device=dev))
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    for v in w:
        v.release()


def test_what_is_still_refused(qm, dev):
    x = torch.empty((0, 64), device=dev)
    for bad in (lambda: qm.quantize_fp8(x, M_stride=-1), lambda: qm.quantize_fp8(torch.ones((1, 64), device=dev), M_stride=0),
                lambda: qm.quantize_fp8(x.double()), lambda: qm.quantize_fp8(x[:, :0]), lambda: qm.swiglu_fp8(x, 33),
                lambda: qm.swiglu_fp8(x, 0), lambda: qm.swiglu_fp8(x, -200), lambda: qm.rmsnorm_fp8(x, torch.ones(63, device=dev), 1e-6)):
        with pytest.raises(qm.QMatmulError):
            bad()
