"""Variants of the e4m3 product (tests/test_fp8_routes.py says which calls take which): pieces of K by the workspace."""
import pytest
import torch

from tests import fp8_plain as P
from tests import test_gpu_fp8 as G

pytestmark = pytest.mark.gpu

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
