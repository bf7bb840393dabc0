"""What the e4m3 products, their producers and the q/k norm + rotation refuse, and what a call of nothing does: through the
C ABI, without a GPU (every check comes before the first device call)."""
import ctypes

import pytest

ARG, SHAPE, TYPE = 1, 2, 3


@pytest.fixture()
def buf():
    b = (ctypes.c_uint8 * (1 << 16))()
    at = ctypes.addressof(b)
    return (at + 255) // 256 * 256, b


def test_sizes(qm):
    lib = qm.load_library()
    assert lib.qmatmul_fp8_weight_bytes(64, 128) == 64 * 128 + 4
    assert lib.qmatmul_fp8_weight_bytes(65, 129) == 128 * 256 + 2 * 4
    assert lib.qmatmul_fp8_weight_bytes(129, 1) == 192 * 128 + 2 * 4
    assert lib.qmatmul_fp8_weight_bytes(0, 128) == 0 and lib.qmatmul_fp8_weight_bytes(16, 0) == 0
    assert lib.qmatmul_fp8_weight_bytes(2 ** 20, 2 ** 20) > 2 ** 40
    assert lib.qmatmul_gemm_fp8_workspace_size(None, 128) == 0


def test_weights(qm, buf):
    lib, (p, _) = qm.load_library(), buf
    h = ctypes.c_void_p(1)
    assert lib.qmatmul_prepare_fp8(None, p, 0, 16, 128, None, ctypes.byref(h)) == ARG
    assert lib.qmatmul_prepare_fp8(p, None, 0, 16, 128, None, ctypes.byref(h)) == ARG
    assert lib.qmatmul_prepare_fp8(p, p, 0, 16, 128, None, None) == ARG
    assert lib.qmatmul_prepare_fp8(p, p, 0, 0, 128, None, ctypes.byref(h)) == SHAPE and h.value is None
    assert lib.qmatmul_prepare_fp8(p, p, 0, 16, -1, None, ctypes.byref(h)) == SHAPE
    assert lib.qmatmul_prepare_fp8(p, p + 2, 0, 16, 128, None, ctypes.byref(h)) == ARG
    assert lib.qmatmul_release_fp8(None) == ARG and lib.qmatmul_fp8_info(None, None, None, None) == ARG


def test_producers(qm, buf):
    lib, (p, _) = qm.load_library(), buf
    q = lambda **k: lib.qmatmul_quantize_fp8(*{**dict(x=p, t=0, ld=256, M=2, Ms=4, K=256, a=p, s=p, st=None), **k}.values())
    assert q(x=None) == ARG and q(a=None) == ARG and q(s=None) == ARG
    assert q(t=2) == TYPE and q(t=8) == TYPE
    assert q(M=5) == SHAPE and q(M=-1) == SHAPE and q(Ms=0, M=0) == SHAPE and q(K=0) == SHAPE and q(ld=255) == SHAPE
    assert q(x=p + 2) == ARG and q(a=p + 8) == ARG and q(s=p + 1) == ARG and q(t=1, x=p + 1) == ARG
    n = lambda **k: lib.qmatmul_rmsnorm_fp8(*{**dict(x=p, t=0, ld=256, w=p, K=256, M=2, Ms=4, eps=1e-6, a=p, s=p, h=None, ldh=0,
                                                     st=None), **k}.values())
    assert n(w=None) == ARG and n(w=p + 2) == ARG and n(h=p, ldh=255) == SHAPE and n(h=p + 1, ldh=256) == ARG and n(M=5) == SHAPE
    g = lambda **k: lib.qmatmul_swiglu_fp8(*{**dict(x=p, t=0, ld=512, F=256, M=2, Ms=4, gelu=0, a=p, s=p, st=None), **k}.values())
    assert g(ld=511) == SHAPE and g(F=0) == SHAPE and g(x=None) == ARG and g(t=9) == TYPE
    assert g(F=0x7fffffff, ld=0x7fffffff) == SHAPE


def test_products(qm, buf):
    """(A weight needs a device: its fields are never reached by these.)"""
    lib, (p, _) = qm.load_library(), buf
    assert lib.qmatmul_gemm_fp8(None, p, p, 1, 1, p, 0, 64, 0, 0, None, 0, None) == ARG
    assert b"null weight" in lib.qmatmul_last_error()


def rope(qm, p, rot=64, adjacent=0, axes=1, turns=0, sections=(0, 0, 0, 0), scale=1.0, **k):
    r = qm.QmRope(rot, adjacent, axes, turns, (ctypes.c_int * 4)(*sections), scale)
    a = dict(x=p, xt=0, ldx=512, T=2, D=64, q_off=0, q_hs=64, HQ=4, k_off=256, k_hs=64, HK=2, wq=None, wk=None, eps=1e-6,
             rope=ctypes.byref(r), pos=p, ps=2, f=p, q=p + 8192, k=p + 16384, ot=0, ldq=256, ldk=128, st=None)
    assert set(k) <= set(a)
    a.update(k)
    return qm.load_library().qmatmul_qk_norm_rope(*a.values())


def test_rotation(qm, buf):
    p, _ = buf
    assert rope(qm, p, T=0) == 0 and rope(qm, p, T=0, x=None, q=None, k=None, pos=None) == 0  # (nothing to do)
    assert rope(qm, p, HQ=0, HK=0) == 0
    assert rope(qm, p, rope=None) == ARG and rope(qm, p, x=None) == ARG and rope(qm, p, q=None) == ARG
    assert rope(qm, p, k=None) == ARG and rope(qm, p, pos=None) == ARG and rope(qm, p, f=None) == ARG
    assert rope(qm, p, xt=2) == TYPE and rope(qm, p, ot=8) == TYPE
    for bad in (dict(D=63), dict(D=0), dict(D=514), dict(T=-1), dict(HQ=-1), dict(HK=-1), dict(rot=65), dict(rot=66), dict(rot=-2),
                dict(axes=0), dict(axes=5), dict(axes=2, sections=(16, 15, 0, 0)), dict(axes=2, sections=(33, -1, 0, 0)),
                dict(axes=2, sections=(16, 16, 0, 0), ps=1), dict(q_off=-1), dict(k_off=-1), dict(q_hs=63), dict(k_hs=60),
                dict(q_off=257), dict(k_off=400), dict(ldq=255), dict(ldk=127), dict(ldx=300), dict(q_hs=2 ** 30)):
        assert rope(qm, p, **bad) == SHAPE, bad
    for bad in (dict(x=p + 2), dict(q=p + 8193), dict(k=p + 16386), dict(pos=p + 1), dict(f=p + 2), dict(wq=p + 1), dict(wk=p + 3),
                dict(xt=1, x=p + 1)):
        assert rope(qm, p, **bad) == ARG, bad


def test_rotation_refuses_overlaps(qm, buf):
    p, _ = buf
    row = 512 * 4
    for bad in (dict(q=p + 4), dict(q=p, ldq=256), dict(q=p, ldq=512, ot=1), dict(k=p, ldk=512), dict(q=p + 1024, ldq=512),
                dict(q=p + 8192, k=p + 8192 + 128, ldq=512, ldk=512),  # the outputs in each other
                dict(q=p + row - 64, ldq=512), dict(q=p, ldq=512, q_hs=128, HQ=2), dict(k=p + 256 * 4, ldk=256)):
        assert rope(qm, p, **bad) == ARG, bad
        assert b"overlap" in qm.load_library().qmatmul_last_error()


def test_rotation_of_one_token_in_place(qm, buf):
    """A single row has no stride: the input's place with another ld is in place all the same, parts of it are overlaps. (Not
    refused as an overlap; without a GPU the call then ends at the device.)"""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on the host buffer")
    p, _ = buf
    for ok in (dict(q=p), dict(k=p + 256 * 4), dict(q=p, k=p + 256 * 4), dict(q=p, ldq=4096)):
        assert rope(qm, p, T=1, **ok) not in (0, ARG, SHAPE, TYPE), ok
    for bad in (dict(q=p + 4), dict(q=p + 256 * 4), dict(q=p, ot=1), dict(q=p, q_hs=128, HQ=2), dict(k=p, ldk=128)):
        assert rope(qm, p, T=1, **bad) == ARG, bad
        assert b"overlap" in qm.load_library().qmatmul_last_error()


def test_normed_copy_beside_its_input(qm, buf):
    """h over x: several work-groups may read a row while one writes its h, so no overlap is taken; rows in turns are none."""
    lib, (p, _) = qm.load_library(), buf
    n = lambda **k: lib.qmatmul_rmsnorm_fp8(*{**dict(x=p, t=0, ld=256, w=p, K=256, M=2, Ms=4, eps=1e-6, a=p, s=p, h=None, ldh=256,  # noqa: E731
                                                     st=None), **k}.values())
    for bad in (dict(h=p), dict(h=p + 4), dict(h=p + 255 * 4), dict(h=p + 256 * 4), dict(h=p + 511 * 4), dict(h=p, ldh=512), dict(h=p, t=1),
                dict(x=p + 2048, h=p + 1024), dict(ld=512, ldh=512, h=p + 255 * 4)):
        assert n(**bad) == ARG, bad
        assert b"overlap" in lib.qmatmul_last_error()
    import torch
    if not torch.cuda.is_available():  # (not refused: the call ends at the device, which is not there)
        for ok in (dict(h=p + 512 * 4), dict(ld=512, ldh=512, h=p + 256 * 4), dict(h=p, x=p + 2048), dict(h=p, M=0)):
            assert n(**ok) not in (0, ARG, SHAPE), ok
