"""Outputs of the e4m3 producers and products over their inputs or over each other: several work-groups share a row, and one would
read what another has written. Refused before any launch; what only lies between the input's rows is not."""
import ctypes

import pytest
import torch

ARG = 1


@pytest.fixture()
def at():
    b = (ctypes.c_uint8 * (1 << 17))()
    yield (ctypes.addressof(b) + 255) // 256 * 256


def is_overlap(qm, st):
    return st == ARG and b"overlap" in qm.load_library().qmatmul_last_error()


def test_rows_and_gates(qm, at):
    """x: two rows of 256 floats; a8: four rows of 256 bytes; asc: 2 x 4 floats."""
    lib, p = qm.load_library(), at
    q = lambda **k: lib.qmatmul_quantize_fp8(*{**dict(x=p, t=0, ld=256, M=2, Ms=4, K=256, a=p + 8192, s=p + 16384, st=None), **k}.values())  # noqa: E731
    g = lambda **k: lib.qmatmul_swiglu_fp8(*{**dict(x=p, t=1, ld=512, F=256, M=2, Ms=4, gelu=0, a=p + 8192, s=p + 16384, st=None), **k}.values())  # noqa: E731
    for f in (q, g):
        for bad in (dict(a=p), dict(s=p), dict(a=p + 2032), dict(s=p + 2044), dict(x=p + 1024, a=p + 16), dict(x=p + 1024, s=p + 996),
                    dict(a=p + 16384, s=p + 16384), dict(a=p + 16384 - 1008), dict(s=p + 8192 + 1020)):
            assert is_overlap(qm, f(**bad)), bad
        row = 4096 * (4 if f is q else 2)  # rows apart: the edges of one, and the gap
        for bad in (dict(ld=4096, a=p + 1024 - 16, s=p + 40000), dict(ld=4096, a=p + 1024, s=p + row - 28)):
            assert is_overlap(qm, f(**bad)), bad
        if not torch.cuda.is_available():  # (not refused: the call ends at the device, which is not there)
            for ok in ({}, dict(a=p + 2048), dict(s=p + 2048), dict(x=p + 1024, a=p), dict(x=p + 32, s=p), dict(M=0, a=p),
                       dict(ld=4096, a=p + 1024, s=p + 40000), dict(ld=4096, a=p + 1024, s=p + row - 32)):
                assert f(**ok) not in (0, ARG, 2, 3), ok


@pytest.mark.gpu
def test_normed_rows(qm, dev):
    lib, buf = qm.load_library(), torch.zeros(1 << 16, dtype=torch.uint8, device=dev)
    p, w = (buf.data_ptr() + 255) // 256 * 256, torch.ones(256, device=dev)
    n = lambda **k: lib.qmatmul_rmsnorm_fp8(*{**dict(x=p, t=0, ld=256, w=w.data_ptr(), K=256, M=2, Ms=4, eps=1e-6, a=p + 8192, s=p + 16384,  # noqa: E731
                                                     h=p + 20480, ldh=256, st=qm._stream(None)), **k}.values())
    for bad in (dict(a=p), dict(s=p), dict(a=p + 2032), dict(s=p + 2044), dict(a=p + 16384), dict(h=p + 8192), dict(h=p + 16384),
                dict(h=p + 8192 - 2044), dict(a=p + 20480), dict(s=p + 20480, h=p + 20480 + 28), dict(h=p)):
        assert is_overlap(qm, n(**bad)), bad
    assert not buf.any()
    assert n() == 0 and n(h=None) == 0 and n(ldh=512, a=p + 20480 + 1024, Ms=2) == 0


@pytest.mark.gpu
def test_products(qm, dev):
    N, K, M = 256, 256, 5
    w = qm.Fp8Weight(torch.zeros((N, K), dtype=torch.uint8, device=dev), torch.ones((2, 2), device=dev))
    lib, buf = qm.load_library(), torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    p = (buf.data_ptr() + 255) // 256 * 256
    f = lambda **k: lib.qmatmul_gemm_fp8(*{**dict(w=w.handle, a=p, s=p + 8192, M=M, Ms=8, C=p + 16384, t=0, ldc=N, off=0, acc=0,  # noqa: E731
                                                  ws=p + 65536, wsb=65536, st=qm._stream(None)), **k}.values())
    row = 4 * N
    for bad in (dict(C=p), dict(C=p + 1276), dict(C=p + 8192 - 5 * row + 4), dict(C=p + 8192), dict(ldc=2048, off=1024, C=p - 4096 + 1276)):
        assert is_overlap(qm, f(**bad)), bad
    assert not buf.any()
    assert f(C=p + 1280) == 0 and f(Ms=4096, C=p + 1280) == 0  # (behind the call's own rows: it may be a part of a longer batch)
    assert f() == 0 and f(ws=None, wsb=0) == 0 and f(ws=p, wsb=0) == 0 and f(ldc=1024, C=p + 8192 + 256) == 0
    assert f(ws=p) == 0 and f(C=p + 65536) == 0  # (so few tokens use no workspace)
    w.release()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [0, 30])
def test_workspaces(qm, dev, t):
    """What the pieces take of the workspace, and no more of it than that."""
    N, K, M = 2048, 9600, 200
    w = qm.Fp8Weight(torch.zeros((N, K), dtype=torch.uint8, device=dev), torch.ones((16, 75), device=dev))
    piece, lib = 4 * M * N, qm.load_library()
    need = lib.qmatmul_gemm_fp8_workspace_size(w.handle, M)
    assert need >= 2 * piece
    buf = torch.zeros(64 << 20, dtype=torch.uint8, device=dev)
    p, size = (buf.data_ptr() + 255) // 256 * 256, 2 if t else 4
    a, s, C, ws = p, p + (2 << 20), p + (3 << 20), p + (8 << 20)
    row = size * N
    f = lambda **k: lib.qmatmul_gemm_fp8(*{**dict(w=w.handle, a=a, s=s, M=M, Ms=M, C=C, t=t, ldc=N, off=0, acc=0, ws=ws, wsb=2 * piece,  # noqa: E731
                                                  st=qm._stream(None)), **k}.values())
    for bad in (dict(ws=a), dict(ws=s), dict(ws=C), dict(ws=C + 199 * row), dict(C=ws), dict(C=ws + 2 * piece - 16), dict(C=ws - 199 * row),
                dict(a=ws + 4096), dict(s=ws + 2 * piece - 4), dict(ldc=4 * N, C=ws - 4 * row)):
        assert is_overlap(qm, f(**bad)), bad
    assert not buf.any()
    assert f() == 0 and f(C=ws + 2 * piece) == 0 and f(C=ws - 200 * row) == 0 and f(ws=C, wsb=piece - 1) == 0
    assert f(wsb=(64 << 20) - (8 << 20) - 256, a=ws + need) == 0
    w.release()
