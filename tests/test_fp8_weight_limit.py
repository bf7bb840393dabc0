"""The largest weight: laid out by a thread for each 16 bytes, of which a grid holds fewer than 2^32 (no GPU: refused before it)."""
import ctypes


def test_weights_of_64_gib_are_refused(qm):
    lib, b = qm.load_library(), (ctypes.c_float * 64)()
    p, h = ctypes.addressof(b), ctypes.c_void_p()
    prepare = lambda rows, K: lib.qmatmul_prepare_fp8(p, p, 1, rows, K, None, ctypes.byref(h))  # noqa: E731
    for rows, K in ((1 << 22, 1 << 14), (1 << 29, 1), (1 << 29, 128), ((1 << 22) - 63, (1 << 14) - 127), (1 << 30, 256)):
        assert prepare(rows, K) == 2 and not h.value, (rows, K)
        assert lib.qmatmul_fp8_weight_bytes(rows, K) > 1 << 36
    import torch
    if not torch.cuda.is_available():  # (not refused: the call ends at the device, which is not there)
        for rows, K in ((64, 1 << 24), ((1 << 22) - 64, 1 << 14), ((1 << 29) - 64, 1)):
            assert prepare(rows, K) not in (0, 1, 2)
