"""Variants of the e4m3 product that no other shape reaches (tests/test_fp8_routes.py says which calls take which): few tokens on
short K, and cuts into 2, 6, 10 and 12 pieces."""
import pytest
import torch

from tests import fp8_plain as P
from tests import test_gpu_fp8 as G

pytestmark = pytest.mark.gpu

SHAPES = [(4200, 130, 1), (512, 1152, 7), (5000, 520, 9), (2975, 2180, 71), (1573, 3727, 67), (1021, 5791, 66), (3797, 1225, 216)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,M", SHAPES)
def test_product(qm, dev, N, K, M, out):
    w, a8, asc, (ref, *sums) = G.make(qm, dev, N, K, M, N + K + M)
    kb = P.up(K, 128) // 128
    for ws in (qm.gemm_fp8_workspace(w, M), torch.empty(64 << 20, dtype=torch.uint8, device=dev)):
        C = qm.gemm_fp8(w, a8, asc, M=M, out=out, ws=ws)
        G.near(C, ref, P.gemm_bound(*sums, kb, out) + P.rounding(out, ref))
    w.release()


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K,M", [(1021, 5791, 66), (2975, 2180, 71)])
def test_fewer_pieces_where_the_workspace_is_smaller(qm, dev, N, K, M, out):
    """Every size from all pieces' to none: the same within the bound, and nothing behind the workspace's end is written."""
    w, a8, asc, (ref, *sums) = G.make(qm, dev, N, K, M, N + K + M)
    bound = P.gemm_bound(*sums, P.up(K, 128) // 128, out) + P.rounding(out, ref)
    piece = M * P.up(N, 64) * 4
    for n in [p * piece - d for p in range(1, 17) for d in (0, 4)] + [4, 256]:
        buf = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device=dev)
        G.near(qm.gemm_fp8(w, a8, asc, M=M, out=out, ws=buf[:n]), ref, bound)
        assert bool((buf[n:] == 0x5A).all())
    w.release()
