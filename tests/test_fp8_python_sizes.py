"""Sizes and strides on their way from Python to the C ABI's 32-bit ints, without a GPU: tensors of the meta device stand for
those of the current GPU, the library's functions are recorded instead of called."""
import pytest
import torch

F32, U8, E4M3 = torch.float32, torch.uint8, torch.float8_e4m3fn
FAR = 2 ** 32  # (modulo which ctypes takes an int)


class Weight:
    """What gemm_fp8 reads of an Fp8Weight."""
    handle, rows, Kp = 1, 200, 384


@pytest.fixture()
def calls(qm, monkeypatch):
    """(function, arguments) of every call of the library."""
    made = []

    def function(name):
        return lambda *a: made.append((name, a)) or 0
    monkeypatch.setattr(qm, "_torch", torch)
    monkeypatch.setattr(qm, "_current_gpu", lambda: -1)  # (what get_device() says of a meta tensor)
    monkeypatch.setattr(qm, "_current_stream", lambda dev: 0)
    monkeypatch.setattr(qm, "_function", function)
    monkeypatch.setattr(qm, "_call", lambda name, *a: made.append((name, a)) or 0)
    return made


def rows(M, W, ld, dtype=F32):
    return torch.empty_strided((M, W), (ld, 1), dtype=dtype, device="meta")


def meta(*shape, dtype=F32):
    return torch.empty(shape, dtype=dtype, device="meta")


def turn(qm, T=3, x=None, q=None, k=None, pos=None, **kw):
    x = meta(T, 384) if x is None else x
    return qm.qk_norm_rope(x, 4, 2, 64, meta(T, dtype=torch.int32) if pos is None else pos, meta(32), q=q, k=k, **kw)


def product(qm, M=3, Ms=16, **kw):
    return qm.gemm_fp8(Weight, meta(Ms, 384, dtype=E4M3), meta(3, Ms), M=M, **kw)


def test_these_calls_are_taken(qm, calls):
    qm.quantize_fp8(rows(3, 256, 2 ** 31 - 1))
    qm.rmsnorm_fp8(rows(3, 256, 260), meta(256), 1e-6)
    qm.swiglu_fp8(rows(3, 512, 512), 256)
    product(qm)
    product(qm, C=rows(3, 200, 2 ** 31 - 1))
    turn(qm, x=rows(3, 384, 2 ** 31 - 1), q=rows(3, 256, 2 ** 31 - 1), k=rows(3, 128, 200))
    turn(qm, pos=torch.empty_strided((2, 3), (2 ** 31 - 1, 1), dtype=torch.int32, device="meta"), sections=(16, 16))
    qm.Fp8Weight(meta(200, 300, dtype=U8), meta(2, 3), stream=0).handle = None
    assert len(calls) == 8 and calls[0][1][2] == 2 ** 31 - 1


@pytest.mark.parametrize("ld", [FAR + 512, 2 ** 31, 2 ** 40 + 600])
def test_far_rows_are_refused(qm, calls, ld):
    """Row strides that a 32-bit int cannot hold: taken modulo 2^32, the rows behind the first would be others."""
    far_pos = torch.empty_strided((2, 3), (ld, 1), dtype=torch.int32, device="meta")
    for bad in (lambda: qm.quantize_fp8(rows(3, 256, ld)), lambda: qm.rmsnorm_fp8(rows(3, 256, ld), meta(256), 1e-6),
                lambda: qm.swiglu_fp8(rows(3, 512, ld), 256), lambda: product(qm, C=rows(3, 200, ld)),
                lambda: product(qm, C=rows(3, 200, ld), ldc=ld), lambda: turn(qm, x=rows(3, 384, ld)), lambda: turn(qm, q=rows(3, 256, ld)),
                lambda: turn(qm, k=rows(3, 128, ld)), lambda: turn(qm, pos=far_pos, sections=(16, 16)),
                lambda: turn(qm, q=torch.empty_strided((3, 4, 64), (ld, 64, 1), device="meta"))):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls


def test_a_single_far_row_is_a_row(qm, calls):
    """A single row's stride says nothing: it is taken, with a stride that the ABI's int holds."""
    ld = FAR + 512
    qm.quantize_fp8(rows(1, 256, ld))
    qm.rmsnorm_fp8(rows(1, 256, ld), meta(256), 1e-6)
    qm.swiglu_fp8(rows(1, 512, ld), 256)
    product(qm, M=1, C=rows(1, 200, ld))
    turn(qm, T=1, x=rows(1, 384, ld), q=rows(1, 256, ld), k=rows(1, 128, ld))
    given = [a[2] for _, a in calls[:3]] + [calls[3][1][7], calls[4][1][2], *calls[4][1][-3:-1]]
    assert given == [256, 256, 512, 200, 384, 256, 128]


def test_far_sizes_are_refused(qm, calls):
    """Counts, offsets and head strides likewise."""
    for bad in (lambda: qm.quantize_fp8(rows(3, 256, 256), M_stride=FAR + 16), lambda: qm.quantize_fp8(rows(FAR + 3, 256, 256)),
                lambda: qm.swiglu_fp8(rows(3, 2 * FAR + 512, 2 * FAR + 512), FAR + 256), lambda: product(qm, M=FAR + 3),
                lambda: product(qm, C=rows(3, FAR + 400, 2 ** 31 - 1), c_off=FAR + 8), lambda: product(qm, C=meta(3, 200), accumulate=FAR),
                lambda: turn(qm, q_off=FAR, x=rows(3, FAR + 384, 2 ** 31 - 1)), lambda: turn(qm, k_off=FAR, x=rows(3, FAR + 384, 2 ** 31 - 1)),
                lambda: turn(qm, q_hs=FAR + 64, k_off=0, x=rows(3, 4 * FAR + 384, 2 ** 31 - 1)),
                lambda: turn(qm, sections=(FAR + 16, 16 - FAR), pos=meta(2, 3, dtype=torch.int32)),
                lambda: qm.Fp8Weight(meta(FAR + 16, 1, dtype=U8), meta((FAR + 16 + 127) // 128, 1), stream=0),
                lambda: qm.gemm_fp8_workspace(Weight, FAR + 64)):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls


def test_no_rows_and_negative_counts(qm, calls):
    """A batch of no rows has empty results, without a call; counts below zero are the library's own errors."""
    for x in (meta(0, 300), meta(0, 300, dtype=torch.bfloat16)):
        for a8, asc, *_ in (qm.quantize_fp8(x), qm.rmsnorm_fp8(x, meta(300), 1e-6, want_h=True), qm.swiglu_fp8(meta(0, 600), 300)):
            assert a8.shape == (0, 384) and asc.shape == (3, 0)
    assert not calls
    qm.quantize_fp8(meta(0, 300), M_stride=4)
    assert calls.pop()[1][3:6] == (0, 4, 300)
    for bad in (lambda: qm.quantize_fp8(meta(3, 300), M_stride=-1), lambda: qm.quantize_fp8(meta(0, 300), M_stride=-1),
                lambda: qm.quantize_fp8(meta(3, 300), M_stride=0), lambda: qm.quantize_fp8(meta(0, 300, dtype=torch.int32)),
                lambda: qm.quantize_fp8(meta(0, 0)), lambda: qm.swiglu_fp8(meta(0, 600), 0), lambda: qm.swiglu_fp8(meta(3, 600), -200),
                lambda: product(qm, M=-1), lambda: product(qm, M=-1, C=meta(3, 200)),
                *(lambda H=H: qm.qk_norm_rope(meta(3, 384), *H, meta(3, dtype=torch.int32), meta(32)) for H in ((-1, 2, 64), (4, -2, 64), (4, 2, -64)))):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls
