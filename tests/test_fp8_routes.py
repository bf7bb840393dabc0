"""The choice among the variants of the e4m3 product (host code of the built library, no GPU): at shapes where each side was measured the
call takes the fastest, the products of tests/test_gpu_fp8.py and tests/test_gpu_fp8_variants.py run every variant that it can take, and a
workspace that is too small for all pieces gets fewer. Times in microseconds, one MI355X."""
import ctypes
import math
import random

import pytest

from tests import test_gpu_fp8, test_gpu_fp8_variants

MOST = 64 << 20  # bytes of workspace that a call uses at most


class Plan(ctypes.Structure):
    _fields_ = [("mt", ctypes.c_int), ("splits", ctypes.c_int), ("rt", ctypes.c_int), ("waves", ctypes.c_int)]


@pytest.fixture(scope="module")
def plan():
    from arcinfer_amd import qmatmul
    f = qmatmul.load_library()._ZN2qm8fp8_planEiiiibm
    f.restype, f.argtypes = Plan, [ctypes.c_int] * 4 + [ctypes.c_bool, ctypes.c_size_t]

    def of(M, N, K, f32, ws=MOST):
        p = f(M, (M + 15) // 16 * 16, N, (K + 127) // 128, f32, ws)
        return (p.mt, p.splits) if p.mt else (0, p.rt, p.waves)
    return of


@pytest.mark.parametrize("M,N,K,f32,want", [
    # few-token kernel
    (32, 9000, 2048, False, (0, 2, 8)),     # 9.8 against 11.0 of the best tiles
    (64, 2560, 2560, False, (0, 1, 8)),     # 8.9, 10.8
    (130, 512, 1024, False, (0, 1, 8)),     # 5.0, 8.0
    (64, 9000, 2048, True, (0, 2, 8)),      # 16.5, 16.7
    (1024, 512, 1024, True, (0, 1, 8)),     # 9.3, 13.2
    # tiles, whole
    (260, 17408, 1024, False, (6, 1)),      # 12.5; the few-token kernel 36.2
    (512, 4096, 4096, False, (4, 1)),       # 20.6; in two pieces 22.5
    (1024, 2560, 2560, False, (4, 1)),      # 15.0; five token tiles 18.9
    (2900, 9000, 2048, False, (7, 1)),      # 63.7; eight token tiles 65.7
    (4096, 5120, 17408, False, (7, 1)),     # 328; eight token tiles 334
    (512, 17408, 1024, True, (5, 1)),       # 26.9; six token tiles 31.6
    (2048, 5120, 5120, True, (6, 1)),       # 110; four token tiles 113
    # tiles, K in pieces
    (64, 5120, 5120, False, (4, 5)),        # 14.2; whole 23.7, few tokens 16.5
    (96, 2048, 12800, False, (4, 10)),      # 16.5; whole 53.0
    (200, 5120, 17408, False, (7, 6)),      # 36.9; four token tiles, whole, 89
    (80, 5120, 17408, True, (5, 12)),       # 31.1; whole 152
    (333, 2048, 12800, True, (4, 10)),      # 32.6; in five 33.9
    (420, 5120, 17408, True, (5, 4)),       # 90.7; whole 155
])
def test_the_fastest_is_taken(plan, M, N, K, f32, want):
    assert plan(M, N, K, f32) == want


def variants(plan, N, K, M):
    for f32 in (True, False):
        p = plan(M, N, K, f32)
        if p[0]:
            yield from ((f32, "tiles", p[0], p[1] > 1), (f32, "pieces", p[1]))
        else:
            yield f32, "few", min(4, (M + 15) // 16), *p[1:]


def test_every_variant_is_tested(plan):
    tested = {v for s in test_gpu_fp8.SHAPES + test_gpu_fp8.VARIANTS + test_gpu_fp8_variants.SHAPES for v in variants(plan, *s)}
    rng = random.Random(0)
    some = lambda a, b: int(math.exp(rng.uniform(math.log(a), math.log(b))))  # noqa: E731
    for i in range(30000):
        shape = some(1, 60000), some(1, 40000), some(1, 300 if i % 2 else 20000)
        missing = set(variants(plan, *shape)) - tested
        assert not missing, (shape, missing)


@pytest.mark.parametrize("f32", [True, False])
def test_work_groups_fit_a_grid(plan, f32):
    """The most rows of a weight, and tokens whose C is within the card's memory: 2^32 threads are not reached."""
    for K in (1, 128, 256, 900, 1100, 2048, 1 << 14, 1 << 24):
        for N in (((1 << 36) - 4096) // ((K + 127) // 128 * 128) // 64 * 64, (1 << 32) // ((K + 127) // 128 * 128)):
            for M in (1, 16, 17, 33, 64, 100, 300, 512, 1000, 1024, 5000, 1 << 20):
                if M * N * (4 if f32 else 2) > 288 << 30:
                    continue
                p = plan(M, N, K, f32)
                if p[0]:
                    groups, waves = (N + 255) // 256 * ((M + 16 * p[0] - 1) // (16 * p[0])) * p[1], 4
                else:
                    mt = min(4, (M + 15) // 16)
                    groups, waves = (N + 63) // 64 * 4 // p[1] * ((M + 16 * mt - 1) // (16 * mt)), p[2]
                assert 0 < groups * 64 * waves < 1 << 32, (M, N, K, p)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("M,N,K", [(66, 1021, 5791), (48, 5120, 17408), (777, 5120, 17408), (333, 5184, 5120), (130, 4096, 4096)])
def test_a_smaller_workspace_has_fewer_pieces(plan, M, N, K, f32):
    piece = 4 * M * ((N + 63) // 64 * 64)
    mt, most = plan(M, N, K, f32)
    assert mt and most > 1 and most * piece <= MOST
    assert plan(M, N, K, f32, most * piece) == (mt, most)
    less = plan(M, N, K, f32, most * piece - 1)  # (fewer pieces, or the few-token kernel where that is faster then)
    assert not less[0] or less[1] < most and (less[1] > 1 or most == 2)
    for ws in range(0, most * piece, piece // 2):
        p = plan(M, N, K, f32, ws)
        assert not p[0] or p[1] == 1 or p[1] * piece <= ws
    assert len(plan(M, N, K, f32, 0)) == 3 or plan(M, N, K, f32, 0)[1] == 1
    assert plan(M, N, K, f32, 1 << 40) == plan(M, N, K, f32)


@pytest.mark.parametrize("M,N,K", [(40, 4096, 4096), (66, 1021, 5791), (48, 5120, 17408), (777, 5120, 17408), (1024, 5120, 17408), (2048, 5120, 17408)])
def test_the_size_that_is_asked_for_holds_all_pieces(plan, M, N, K):
    from arcinfer_amd import qmatmul
    size = qmatmul.load_library()._ZN2qm19fp8_workspace_bytesEiii
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_int] * 3
    n = size(M, N, K // 128 + (K % 128 > 0))
    assert n <= MOST
    for f32 in (True, False):
        assert plan(M, N, K, f32, n) == plan(M, N, K, f32)
