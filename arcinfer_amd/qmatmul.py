"""ctypes binding of libqmatmul.so (include/qmatmul.h) and torch-tensor conveniences.

The library is the product: this module only passes device pointers and sizes through the C ABI. It raises
QMatmulError for any non-zero status, and refuses to run when the library is not built (there is no fallback).
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libqmatmul.so")

QM_OK = 0
STATUS_NAMES = {0: "QM_OK", 1: "QM_ERR_ARG", 2: "QM_ERR_SHAPE", 3: "QM_ERR_TYPE", 4: "QM_ERR_HIP",
                5: "QM_ERR_NOMEM", 6: "QM_ERR_WORKSPACE"}

# every function include/qmatmul.h declares: (name, restype, argtypes)
_c = ctypes
_P = _c.c_void_p
_I = _c.c_int
_Z = _c.c_size_t
SIGNATURES = [
    ("qmatmul_init", _I, []),
    ("qmatmul_last_error", _c.c_char_p, []),
    ("qmatmul_sb_bytes", _Z, [_I]),
    ("qmatmul_weight_bytes", _Z, [_I, _I, _I]),
    ("qmatmul_prepare_weight", _I, [_I, _P, _I, _I, _I, _P, _c.POINTER(_P)]),
    ("qmatmul_release_weight", _I, [_P]),
    ("qmatmul_weight_info", _I, [_P, _c.POINTER(_I), _c.POINTER(_I), _c.POINTER(_I)]),
    ("qmatmul_quantize_act", _I, [_P, _I, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_quantize_act_ex", _I, [_P, _I, _I, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_gemv", _I, [_P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P]),
    ("qmatmul_gemm", _I, [_P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P]),
    ("qmatmul_gemm_ex", _I, [_P, _P, _P, _P, _I, _I, _I, _P, _I, _I, _I, _P]),
    ("qmatmul_gemm_noalloc", _I, [_P, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P]),
    ("qmatmul_gemm_workspace_size", _Z, [_P, _I]),
    ("qmatmul_gemm_ws", _I, [_P, _P, _P, _P, _I, _I, _I, _P, _I, _I, _I, _P, _Z, _P]),
    ("qmatmul_moe_workspace_size", _Z, [_I, _I, _I, _I, _I]),
    ("qmatmul_moe_route", _I, [_P, _I, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_moe_grouped", _I, [_P, _P, _P, _I, _P, _I, _I, _I, _P, _P, _I, _P, _I, _P, _Z, _P]),
    ("qmatmul_moe_grouped_ex", _I, [_P, _P, _P, _I, _P, _I, _I, _I, _P, _P, _I, _P, _P, _I, _I, _P, _I, _P, _Z, _P]),
    ("qmatmul_moe_ws_layout", _I, [_I, _I, _I, _I, _I, _P]),
    ("qmatmul_gemv_blocksums", _I, [_P, _P, _P, _I, _I, _P, _P, _P]),
    ("qmatmul_gemm_blocksums", _I, [_P, _P, _I, _I, _P, _P]),
    ("qmatmul_rmsnorm_quant", _I, [_P, _I, _P, _I, _I, _I, _c.c_float, _P, _P, _P, _P, _I, _P]),
    ("qmatmul_swiglu_quant", _I, [_P, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_add_norm_quant", _I, [_P, _P, _P, _I, _c.c_float, _c.c_float, _P, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_rmsnorm_quant_ex", _I, [_P, _I, _P, _I, _I, _I, _c.c_float, _I, _P, _P, _P, _P, _I, _P]),
    ("qmatmul_swiglu_quant_ex", _I, [_P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_add_norm_quant_ex", _I, [_P, _P, _P, _I, _c.c_float, _c.c_float, _P, _I, _I, _I, _P, _P, _P, _P]),
    ("qmatmul_fp8_weight_bytes", _Z, [_I, _I]),
    ("qmatmul_prepare_fp8", _I, [_P, _P, _I, _I, _I, _P, _c.POINTER(_P)]),
    ("qmatmul_release_fp8", _I, [_P]),
    ("qmatmul_fp8_info", _I, [_P, _c.POINTER(_I), _c.POINTER(_I), _c.POINTER(_I)]),
    ("qmatmul_quantize_fp8", _I, [_P, _I, _I, _I, _I, _I, _P, _P, _P]),
    ("qmatmul_rmsnorm_fp8", _I, [_P, _I, _I, _P, _I, _I, _I, _c.c_float, _P, _P, _P, _I, _P]),
    ("qmatmul_swiglu_fp8", _I, [_P, _I, _I, _I, _I, _I, _I, _P, _P, _P]),
    ("qmatmul_gemm_fp8_workspace_size", _Z, [_P, _I]),
    ("qmatmul_gemm_fp8", _I, [_P, _P, _P, _I, _I, _P, _I, _I, _I, _I, _P, _Z, _P]),
    ("qmatmul_qk_norm_rope", _I, [_P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _c.c_float, _P, _P, _I, _P, _P, _P,
                                  _I, _I, _I, _P]),
    ("qmatmul_gguf_open", _I, [_c.c_char_p, _c.POINTER(_P)]),
    ("qmatmul_gguf_close", _I, [_P]),
    ("qmatmul_gguf_tensor_count", _I, [_P, _c.POINTER(_I)]),
    ("qmatmul_gguf_find_tensor", _I, [_P, _c.c_char_p, _c.POINTER(_I)]),
    ("qmatmul_gguf_tensor_info", _I, [_P, _I, _c.POINTER(_c.c_char_p), _c.POINTER(_I), _c.POINTER(_I),
                                      _c.POINTER(_c.c_uint64), _c.POINTER(_P), _c.POINTER(_c.c_uint64)]),
    ("qmatmul_gguf_get_int", _I, [_P, _c.c_char_p, _c.POINTER(_c.c_int64)]),
    ("qmatmul_gguf_get_float", _I, [_P, _c.c_char_p, _c.POINTER(_c.c_double)]),
    ("qmatmul_gguf_get_str", _I, [_P, _c.c_char_p, _c.POINTER(_c.c_char_p)]),
]


class QMatmulError(RuntimeError):
    def __init__(self, fn, status, msg):
        super().__init__(f"{fn}: {STATUS_NAMES.get(status, status)}: {msg}")
        self.status = status


class MoeWsLayout(ctypes.Structure):
    _fields_ = [(n, ctypes.c_size_t) for n in
                ("ids", "wts", "counts", "cursor", "tstart", "tiles", "stok", "swt", "inv", "hq", "hsc", "y",
                 "hf", "total")] + [("slots", ctypes.c_int), ("max_tiles", ctypes.c_int), ("tile_rows", ctypes.c_int)]


_lib = None


def load_library(path=LIB_PATH):
    """Loads libqmatmul.so (built in-tree by arcinfer_amd.build); raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is not built: run `python -m arcinfer_amd.build` (there is no fallback path)")
    # One HIP runtime per process: torch ships its own libamdhip64.so.7 and loads it under another file name, so
    # it must be loaded first; the library's libamdhip64.so.7 dependency then binds to that copy (by soname)
    # instead of bringing in /opt/rocm's as a second runtime that would not know torch's memory and streams.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(path)
    for name, res, args in SIGNATURES:
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _lib = lib
    return lib


def _call(name, *args):
    lib = load_library()
    st = getattr(lib, name)(*args)
    if st != QM_OK:
        raise QMatmulError(name, st, lib.qmatmul_last_error().decode())
    return st


# ---- torch helpers ------------------------------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_raw_stream = None  # device -> torch's current stream there as a number, without the Stream object (2.5 us a call)


def _current_stream(dev):
    global _raw_stream
    if _raw_stream is None:
        import torch
        torch.cuda.current_stream()  # (starts torch's GPU side)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(dev)


def _stream(stream):
    if stream is not None:
        return ctypes.c_void_p(stream)
    import torch
    return ctypes.c_void_p(_current_stream(torch.cuda.current_device()))


class QWeight:
    """A prepared weight (qm_weight*) from GGUF bytes: a uint8 tensor (device or CPU) or a numpy array. K is the raw
    row length; Q8_0 / Q4_0 / IQ4_NL / Q2_0 rows of K % 256 != 0 are padded with zero blocks, and self.K is then the
    prepared (padded) length, self.K_raw the given one."""

    def __init__(self, qtype, raw, rows, K, stream=None):
        import numpy as np
        import torch
        self.qtype, self.rows, self.K = int(qtype), int(rows), int(K)
        self.K_raw = self.K
        h = ctypes.c_void_p()
        if isinstance(raw, np.ndarray):
            raw = np.ascontiguousarray(raw)
            _call("qmatmul_prepare_weight", self.qtype, ctypes.c_void_p(raw.ctypes.data), 0, self.rows, self.K,
                  _stream(stream), ctypes.byref(h))
        else:
            assert isinstance(raw, torch.Tensor) and raw.is_contiguous()
            _call("qmatmul_prepare_weight", self.qtype, _ptr(raw), 1 if raw.is_cuda else 0, self.rows, self.K,
                  _stream(stream), ctypes.byref(h))
        self.handle = h
        k = ctypes.c_int()
        _call("qmatmul_weight_info", h, None, None, ctypes.byref(k))
        self.K = k.value

    @property
    def nbytes(self):
        return load_library().qmatmul_weight_bytes(self.qtype, self.rows, self.K)

    def release(self):
        if self.handle:
            _call("qmatmul_release_weight", self.handle)
            self.handle = None

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.qmatmul_release_weight(self.handle)
                self.handle = None
        except Exception:
            pass


def quantize_act(x, M_stride=None, stream=None, act32=True):
    """x f32 [M, K] (cuda) -> (aq int8 [M_stride, K], asc f32 [K/32, M_stride], absum int16 [K/16, M_stride]);
    act32=False: per-256 scales, asc [K/256, M_stride] (qmatmul_quantize_act_ex)."""
    M, K = x.shape
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _out_acts(Ms, K, x.device, act32)
    if act32:
        _call("qmatmul_quantize_act", _ptr(x), x.stride(0), M, Ms, K, _ptr(aq), _ptr(asc), _ptr(absum), _stream(stream))
    else:
        _call("qmatmul_quantize_act_ex", _ptr(x), x.stride(0), M, Ms, K, 0, _ptr(aq), _ptr(asc), _ptr(absum),
              _stream(stream))
    return aq, asc, absum


def gemv(w, aq, asc, absum, T=1, C=None, ldc=None, c_off=0, accumulate=0, stream=None):
    import torch
    Ms = aq.shape[0]
    if C is None:
        C = torch.empty((T, w.rows), dtype=torch.float32, device=aq.device)
        ldc = w.rows
    _call("qmatmul_gemv", w.handle, _ptr(aq), _ptr(asc), _ptr(absum), Ms, T, _ptr(C),
          w.rows if ldc is None else ldc, c_off, accumulate, _stream(stream))
    return C


def gemm(w, aq, asc, absum, M=None, C=None, ldc=None, c_off=0, accumulate=0, stream=None, noalloc=False, act32=True):
    """qmatmul_gemm (noalloc=True: qmatmul_gemm_noalloc, the entry point that allocates no device memory;
    act32=False: qmatmul_gemm_ex with per-256 activation scales)."""
    import torch
    Ms = aq.shape[0]
    M = Ms if M is None else M
    if C is None:
        C = torch.empty((M, w.rows), dtype=torch.float32, device=aq.device)
        ldc = w.rows
    if not act32:
        if noalloc:
            raise ValueError("qmatmul_gemm_noalloc takes per-32 activation scales only")
        _call("qmatmul_gemm_ex", w.handle, _ptr(aq), _ptr(asc), _ptr(absum), M, Ms, 0, _ptr(C),
              w.rows if ldc is None else ldc, c_off, accumulate, _stream(stream))
        return C
    _call("qmatmul_gemm_noalloc" if noalloc else "qmatmul_gemm", w.handle, _ptr(aq), _ptr(asc), _ptr(absum), M, Ms, _ptr(C),
          w.rows if ldc is None else ldc, c_off, accumulate, _stream(stream))
    return C


def gemm_workspace_size(w, M):
    return load_library().qmatmul_gemm_workspace_size(w.handle, M)


def gemm_ws(w, aq, asc, absum, ws, M=None, C=None, ldc=None, c_off=0, accumulate=0, stream=None, act32=True):
    """qmatmul_gemm_ws: the prompt GEMM with a caller-owned workspace ws (a uint8 device tensor, or None when
    gemm_workspace_size(w, M) is 0)."""
    import torch
    Ms = aq.shape[0]
    M = Ms if M is None else M
    if C is None:
        C = torch.empty((M, w.rows), dtype=torch.float32, device=aq.device)
        ldc = w.rows
    _call("qmatmul_gemm_ws", w.handle, _ptr(aq), _ptr(asc), _ptr(absum), M, Ms, int(act32), _ptr(C),
          w.rows if ldc is None else ldc, c_off, accumulate, _ptr(ws), 0 if ws is None else ws.numel(),
          _stream(stream))
    return C


def gemv_blocksums(w, aq, absum, T=1, stream=None):
    import torch
    nb = w.K // 32
    isum = torch.empty((T, w.rows, nb), dtype=torch.int32, device=aq.device)
    msum = torch.empty((T, w.rows, nb), dtype=torch.int32, device=aq.device) if w.qtype in (12, 13, 10) else None
    _call("qmatmul_gemv_blocksums", w.handle, _ptr(aq), _ptr(absum), aq.shape[0], T, _ptr(isum), _ptr(msum),
          _stream(stream))
    return isum, msum


def gemm_blocksums(w, aq, M=None, stream=None):
    import torch
    M = aq.shape[0] if M is None else M
    isum = torch.empty((M, w.rows, w.K // 32), dtype=torch.int32, device=aq.device)
    _call("qmatmul_gemm_blocksums", w.handle, _ptr(aq), M, aq.shape[0], _ptr(isum), _stream(stream))
    return isum


def moe_route(logits, NU, NE=None, stream=None):
    import torch
    T, ldl = logits.shape
    NE = ldl if NE is None else NE
    ids = torch.empty((T, NU), dtype=torch.int32, device=logits.device)
    wts = torch.empty((T, NU), dtype=torch.float32, device=logits.device)
    counts = torch.empty((NE,), dtype=torch.int32, device=logits.device)
    _call("qmatmul_moe_route", _ptr(logits), ldl, T, NE, NU, _ptr(ids), _ptr(wts), _ptr(counts), _stream(stream))
    return ids, wts, counts


def moe_ws_layout(T, NE, NU, E, F):
    L = MoeWsLayout()
    _call("qmatmul_moe_ws_layout", T, NE, NU, E, F, ctypes.byref(L))
    return L


def moe_workspace(T, NE, NU, E, F, device="cuda"):
    import torch
    n = load_library().qmatmul_moe_workspace_size(T, NE, NU, E, F)
    return torch.empty((n,), dtype=torch.uint8, device=device)


def moe_grouped(gate, up, down, NE, logits, NU, aq, asc, x, ws, T=None, accumulate=0, stream=None, escale=None,
                sh=None, sh_gated=True):
    """qmatmul_moe_grouped, or qmatmul_moe_grouped_ex when escale [NE] or a shared expert's output sh [T, E] is
    given (sh_gated: gate it with sigmoid(logits[t, NE]), logits then having NE + 1 columns)."""
    T = logits.shape[0] if T is None else T
    if escale is None and sh is None:
        _call("qmatmul_moe_grouped", gate.handle, up.handle, down.handle, NE, _ptr(logits), logits.stride(0), T, NU,
              _ptr(aq), _ptr(asc), aq.shape[0], _ptr(x), accumulate, _ptr(ws), ws.numel(), _stream(stream))
    else:
        _call("qmatmul_moe_grouped_ex", gate.handle, up.handle, down.handle, NE, _ptr(logits), logits.stride(0), T,
              NU, _ptr(aq), _ptr(asc), aq.shape[0], _ptr(escale), _ptr(sh), 0 if sh is None else sh.stride(0),
              1 if sh_gated else 0, _ptr(x), accumulate, _ptr(ws), ws.numel(), _stream(stream))
    return x


def _out_acts(Ms, K, dev, act32=True):
    import torch
    return (torch.empty((Ms, K), dtype=torch.int8, device=dev),
            torch.empty((K // (32 if act32 else 256), Ms), dtype=torch.float32, device=dev),
            torch.empty((K // 16, Ms), dtype=torch.int16, device=dev))


def rmsnorm_quant(x, w, eps, M_stride=None, want_h=False, stream=None, act32=True):
    """x f32 [M, K] (cuda), w [K] -> (aq, asc, absum, h or None); act32=False: per-256 scales."""
    import torch
    M, K = x.shape
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _out_acts(Ms, K, x.device, act32)
    h = torch.empty((Ms, K), dtype=torch.float32, device=x.device) if want_h else None
    _call("qmatmul_rmsnorm_quant_ex", _ptr(x), x.stride(0), _ptr(w), K, M, Ms, float(eps), int(act32), _ptr(aq),
          _ptr(asc), _ptr(absum), _ptr(h), K, _stream(stream))
    return aq, asc, absum, h


def swiglu_quant(gu, F, fused=False, gelu=False, M_stride=None, stream=None, act32=True):
    M = gu.shape[0]
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _out_acts(Ms, F, gu.device, act32)
    _call("qmatmul_swiglu_quant_ex", _ptr(gu), gu.stride(0), F, M, Ms, int(fused), int(gelu), int(act32), _ptr(aq),
          _ptr(asc), _ptr(absum), _stream(stream))
    return aq, asc, absum


def add_norm_quant(x, t, w, eps, s, w2=None, M_stride=None, stream=None, act32=True):
    """Updates x in place; returns (aq, asc, absum)."""
    M, K = x.shape
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _out_acts(Ms, K, x.device, act32)
    _call("qmatmul_add_norm_quant_ex", _ptr(x), _ptr(t), _ptr(w), K, float(eps), float(s), _ptr(w2), M, Ms,
          int(act32), _ptr(aq), _ptr(asc), _ptr(absum), _stream(stream))
    return aq, asc, absum


# ---- 8-bit floating point products, query and key heads --------------------------------------------------------------
_DTYPES = {}  # torch dtype -> qm_dtype (filled on first use: torch is imported late)


def _dtype(t):
    d = _DTYPES.get(t)
    if d is None:
        import torch
        _DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
        if t not in _DTYPES:
            raise QMatmulError("dtype", 3, f"{t}: float32, float16 or bfloat16 rows")
        d = _DTYPES[t]
    return d


def _refuse(fn, what):
    raise QMatmulError(fn, 1, what)


_functions = {}


def _function(name):
    """The library's function, bound once: these calls are short, and what Python does for them is most of their time."""
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(load_library(), name)
    return f


def _done(fn, status):
    if status != QM_OK:
        raise QMatmulError(fn, status, load_library().qmatmul_last_error().decode())


_torch = None  # (an import statement in a function is 0.3 us a call, and these calls take about ten)


def _current_gpu():
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch.cuda.current_device()


def _check_rows(fn, name, t, dim, dev):
    """t is on GPU `dev`, of `dim` dimensions where dim is given, its last one contiguous."""
    if t.get_device() == dev and (not dim or t.dim() == dim) and t.stride(-1) == 1:
        return
    if t.get_device() != dev:
        _refuse(fn, f"{name} is on {t.device}, not on the current GPU")
    if dim and t.dim() != dim:
        _refuse(fn, f"{name} has {t.dim()} dimensions, not {dim}")
    if t.numel() and t.shape[-1] != 1:
        _refuse(fn, f"the last dimension of {name} is not contiguous")


_INT_MAX = 0x7fffffff


def _sizes(fn, *v):
    """The library's sizes are 32-bit ints, and ctypes takes a larger number modulo 2^32. (Calls test (a | b | ...) >> 31 first:
    0 where none is negative or too large, in a fifth of the time.)"""
    if max(v) > _INT_MAX or min(v) < -_INT_MAX:
        _refuse(fn, f"sizes, offsets and strides are of 32 bits: {[i for i in v if abs(i) > _INT_MAX]}")


def _stride_of(ld, length, rows):
    """A row stride in elements; of a single row, whose stride says nothing, one that holds the row."""
    return ld if rows > 1 or length <= ld <= _INT_MAX else length


def _row_stride(t):
    """The row stride of a matrix in elements."""
    ld = t.stride(0)
    return ld if t.size(0) > 1 else _stride_of(ld, t.size(1), 1)


class Fp8Weight:
    """A prepared e4m3 weight (qm_fp8_weight*): w8 torch.float8_e4m3fn (or its bytes as uint8) [rows, K], scales float32
    [ceil(rows / 128), ceil(K / 128)], both on the current GPU or both on the CPU. Kp: the activations' row length."""

    def __init__(self, w8, scales, stream=None):
        import torch
        fn = "qmatmul_prepare_fp8"
        self.handle = None
        if w8.dtype not in (torch.float8_e4m3fn, torch.uint8) or w8.dim() != 2 or not w8.is_contiguous():
            _refuse(fn, f"w8 {tuple(w8.shape)} {w8.dtype}: a contiguous matrix of float8_e4m3fn (or its bytes)")
        self.rows, self.K = w8.shape
        self.Kp = (self.K + 127) // 128 * 128
        _sizes(fn, self.rows, self.K)
        if (scales.dtype != torch.float32 or not scales.is_contiguous()
                or tuple(scales.shape) != ((self.rows + 127) // 128, self.Kp // 128)):
            _refuse(fn, f"scales {tuple(scales.shape)} {scales.dtype}: contiguous float32, one for each 128 x 128 block")
        if w8.device != scales.device:
            _refuse(fn, "w8 and scales are on different devices")
        if w8.is_cuda:
            _check_rows(fn, "w8", w8, 2, _current_gpu())
        h = ctypes.c_void_p()
        _call(fn, _ptr(w8), _ptr(scales), 1 if w8.is_cuda else 0, self.rows, self.K, _stream(stream), ctypes.byref(h))
        self.handle = h

    @property
    def nbytes(self):
        return load_library().qmatmul_fp8_weight_bytes(self.rows, self.K)

    def release(self):
        if self.handle:
            h, self.handle = self.handle, None
            _call("qmatmul_release_fp8", h)

    def __del__(self):
        try:
            if self.handle and _lib is not None:
                _lib.qmatmul_release_fp8(self.handle)
                self.handle = None
        except Exception:
            pass


def _out_fp8(fn, x, M, K, M_stride):
    """(M_stride, ldx, a8, asc) of a producer's rows x; where M_stride is 0 there is nothing to call for."""
    Ms, ldx = M if M_stride is None else M_stride, x.stride(0) if M > 1 else _row_stride(x)
    if (M | Ms | K | ldx) >> 31 or Ms == 0:
        _sizes(fn, M, Ms, K, ldx)
        _dtype(x.dtype)
        if Ms < M or K < 1:
            _refuse(fn, f"M {M}, M_stride {Ms}, K {K}")
    Kp = (K + 127) // 128 * 128
    return (Ms, ldx, x.new_empty((Ms, Kp), dtype=_torch.float8_e4m3fn), x.new_empty((Kp // 128, Ms), dtype=_torch.float32))


def quantize_fp8(x, M_stride=None, stream=None):
    """x [M, K] (float32, float16 or bfloat16, rows of any stride) -> (a8 float8_e4m3fn [M_stride, Kp], asc float32
    [Kp / 128, M_stride]), Kp = K rounded up to 128."""
    fn = "qmatmul_quantize_fp8"
    dev = _current_gpu()
    _check_rows(fn, "x", x, 2, dev)
    M, K = x.shape
    Ms, ldx, a8, asc = _out_fp8(fn, x, M, K, M_stride)
    if Ms == 0:
        return a8, asc
    st = _function(fn)(x.data_ptr(), _dtype(x.dtype), ldx, M, Ms, K, a8.data_ptr(), asc.data_ptr(),
                       _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return a8, asc


def rmsnorm_fp8(x, w, eps, M_stride=None, want_h=False, stream=None):
    """x [M, K], w float32 [K] -> (a8, asc, h float32 [M, K] or None)."""
    fn = "qmatmul_rmsnorm_fp8"
    dev = _current_gpu()
    torch = _torch
    _check_rows(fn, "x", x, 2, dev)
    _check_rows(fn, "w", w, 1, dev)
    M, K = x.shape
    if w.dtype != torch.float32 or w.numel() != K:
        _refuse(fn, f"w {tuple(w.shape)} {w.dtype}: float32, one for each of {K} columns")
    Ms, ldx, a8, asc = _out_fp8(fn, x, M, K, M_stride)
    h = x.new_empty((M, K), dtype=torch.float32) if want_h else None
    if Ms == 0:
        return a8, asc, h
    st = _function(fn)(x.data_ptr(), _dtype(x.dtype), ldx, w.data_ptr(), K, M, Ms, eps, a8.data_ptr(),
                       asc.data_ptr(), h.data_ptr() if want_h and M else None, K,
                       _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return a8, asc, h


def swiglu_fp8(gu, F, gelu=False, M_stride=None, stream=None):
    """gu [M, 2 F] (gate then up) -> (a8, asc) of silu(gate) * up, or gelu_tanh(gate) * up."""
    fn = "qmatmul_swiglu_fp8"
    dev = _current_gpu()
    _check_rows(fn, "gu", gu, 2, dev)
    M = gu.size(0)
    if gu.size(1) < 2 * F:
        _refuse(fn, f"rows of {gu.shape[1]} elements hold no gate and up of {F}")
    Ms, ldg, a8, asc = _out_fp8(fn, gu, M, F, M_stride)
    if Ms == 0:
        return a8, asc
    st = _function(fn)(gu.data_ptr(), _dtype(gu.dtype), ldg, F, M, Ms, 1 if gelu else 0, a8.data_ptr(),
                       asc.data_ptr(), _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return a8, asc


def gemm_fp8_workspace(w, M):
    """A workspace for products of M tokens with w (None where they need none). Its size does not grow with M: for calls of several
    M take the largest, or 64 MiB, which serves every call."""
    import torch
    _sizes("qmatmul_gemm_fp8_workspace_size", M)
    n = load_library().qmatmul_gemm_fp8_workspace_size(w.handle, M)
    return torch.empty((n,), dtype=torch.uint8, device="cuda") if n else None


def gemm_fp8(w, a8, asc, M=None, C=None, ldc=None, c_off=0, accumulate=0, out=None, ws=None, stream=None):
    """C [M, rows] (op)= the product of activations (a8, asc) with an Fp8Weight. out: the type of a new C (float32 unless
    given). C: a matrix of its own row stride unless ldc is given."""
    fn = "qmatmul_gemm_fp8"
    dev = _current_gpu()
    torch = _torch
    _check_rows(fn, "a8", a8, 2, dev)
    _check_rows(fn, "asc", asc, 2, dev)
    Ms, Kp = a8.shape
    if M is None:
        M = Ms
    if w.handle is None:
        _refuse(fn, "the weight was released")
    if Kp != w.Kp or a8.dtype not in (torch.float8_e4m3fn, torch.uint8) or not a8.is_contiguous():
        _refuse(fn, f"a8 {tuple(a8.shape)} {a8.dtype}: contiguous rows of {w.Kp} float8_e4m3fn (or their bytes)")
    if asc.dtype != torch.float32 or asc.shape[0] != Kp // 128 or asc.shape[1] != Ms or not asc.is_contiguous():
        _refuse(fn, f"asc {tuple(asc.shape)} {asc.dtype}: contiguous float32 [{Kp // 128}, {Ms}]")
    if (M | Ms | c_off | accumulate) >> 31:
        _sizes(fn, M, Ms, c_off, accumulate)
        if M < 0:
            _refuse(fn, f"M {M}")
    if C is None:
        if accumulate or c_off or ldc is not None:
            _refuse(fn, "accumulate, c_off and ldc need a C")
        C = asc.new_empty((M, w.rows), dtype=out)
        ldc = w.rows
    else:
        _check_rows(fn, "C", C, 2, dev)
        if out is not None and out != C.dtype:
            _refuse(fn, f"out {out} is not C's type")
        own = ldc is None
        if own:
            ldc = _row_stride(C)
        if M > 0 and (M > C.size(0) or c_off + w.rows > C.size(1) if own else
                      (M - 1) * ldc + c_off + w.rows > (C.size(0) - 1) * C.stride(0) + C.size(1)):
            _refuse(fn, f"C {tuple(C.shape)} does not hold {M} rows of {w.rows} from column {c_off} on")
        if ldc >> 31:
            _sizes(fn, ldc)
    if ws is None:
        ws_ptr, ws_bytes = None, 0
    else:
        _check_rows(fn, "ws", ws, 1, dev)
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    st = _function(fn)(w.handle, a8.data_ptr(), asc.data_ptr(), M, Ms, C.data_ptr(), _dtype(C.dtype), ldc, c_off, accumulate,
                       ws_ptr, ws_bytes, _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return C


class QmRope(ctypes.Structure):
    _fields_ = [("rot", _I), ("adjacent", _I), ("axes", _I), ("turns", _I), ("sections", _I * 4), ("scale", _c.c_float)]


def qk_norm_rope(x, HQ, HK, D, pos, inv_freq, wq=None, wk=None, eps=1e-6, adjacent=False, sections=None, turns=False,
                 scale=1.0, q_off=0, q_hs=None, k_off=None, k_hs=None, q=None, k=None, out=None, stream=None):
    """RMS norm (wq, wk float32 [D]; None: no norm) and rotation of the query and key heads in rows x [T, ldx]: query head h at
    column q_off + h * q_hs (D unless given), key head h at k_off + h * k_hs (k_off: behind the query heads unless given).
    pos int32 [T], or [axes, T] with sections (pairs of each axis, behind one another or in turns); inv_freq float32
    [rot / 2]: its length says how many elements of a head turn. Returns (q [T, HQ, D], k [T, HK, D]) of type out (that of
    a given q or k, else x's), or writes the q and k given (matrices [T, HQ * D] or [T, HQ, D] of any row stride; views of x for
    in place)."""
    fn = "qmatmul_qk_norm_rope"
    dev = _current_gpu()
    torch = _torch
    f32 = torch.float32
    axes, half = 1 if pos.dim() == 1 else pos.size(0), inv_freq.numel()
    T = x.size(0)
    # (one test for what is nearly always so; what fails it is named, or allowed, below)
    if not (x.get_device() == dev and x.dim() == 2 and x.stride(1) == 1
            and pos.get_device() == dev and pos.dtype is torch.int32 and pos.size(-1) == T and pos.stride(-1) == 1 and pos.dim() < 3
            and inv_freq.get_device() == dev and inv_freq.dtype is f32 and inv_freq.dim() == 1 and inv_freq.stride(0) == 1
            and (wq is None or (wq.get_device() == dev and wq.dtype is f32 and wq.dim() == 1 and wq.size(0) == D and wq.stride(0) == 1))
            and (wk is None or (wk.get_device() == dev and wk.dtype is f32 and wk.dim() == 1 and wk.size(0) == D and wk.stride(0) == 1))):
        _check_rows(fn, "x", x, 2, dev)
        _check_rows(fn, "inv_freq", inv_freq, 1, dev)
        _check_rows(fn, "pos", pos, None, dev)
        if pos.dtype != torch.int32 or pos.dim() not in (1, 2) or pos.shape[-1] != T:
            _refuse(fn, f"pos {tuple(pos.shape)} {pos.dtype}: int32, one column for each of {T} tokens")
        if inv_freq.dtype != f32:
            _refuse(fn, f"inv_freq {inv_freq.dtype}: float32")
        for w in (wq, wk):
            if w is not None:
                _check_rows(fn, "wq or wk", w, 1, dev)
                if w.dtype != f32 or w.numel() != D:
                    _refuse(fn, f"wq or wk {tuple(w.shape)} {w.dtype}: float32 [{D}]")
    width = x.size(1)
    if sections is None:
        sections = (half,)
    if len(sections) != axes or axes > 4 or sum(sections) != half:
        _refuse(fn, f"sections {sections}: one for each of {axes} axes (at most 4), their sum {half}")
    rope = QmRope(2 * half, adjacent, axes, turns, tuple(sections), scale)
    if q_hs is None:
        q_hs = D
    if k_hs is None:
        k_hs = D
    if k_off is None:
        k_off = q_off + HQ * q_hs
    ldx, ps = x.stride(0) if T > 1 else _row_stride(x), pos.stride(0) if axes > 1 else T
    # (sections of none below zero are within their sum)
    if (T | D | HQ | HK | ldx | ps | q_off | q_hs | k_off | k_hs | 2 * half) >> 31 or (axes > 1 and min(sections) < 0):
        _sizes(fn, T, D, HQ, HK, ldx, ps, q_off, q_hs, k_off, k_hs, 2 * half, *sections)
        if min(D, HQ, HK) < 0:
            _refuse(fn, f"D {D}, HQ {HQ}, HK {HK}")
    if (HQ and q_off + (HQ - 1) * q_hs + D > width) or (HK and k_off + (HK - 1) * k_hs + D > width):
        _refuse(fn, f"rows of {width} elements do not hold the heads")
    if out is None:
        out = q.dtype if q is not None else k.dtype if k is not None else x.dtype
    if q is None:
        q, ldq = x.new_empty((T, HQ, D), dtype=out), HQ * D
    else:
        ldq = _head_rows(fn, "q", q, T, HQ, D, out, dev)
    if k is None:
        k, ldk = x.new_empty((T, HK, D), dtype=out), HK * D
    else:
        ldk = _head_rows(fn, "k", k, T, HK, D, out, dev)
    st = _function(fn)(x.data_ptr(), _dtype(x.dtype), ldx, T, D, q_off, q_hs, HQ, k_off, k_hs, HK,
                       None if wq is None else wq.data_ptr(), None if wk is None else wk.data_ptr(), eps, ctypes.byref(rope),
                       pos.data_ptr(), ps, inv_freq.data_ptr(), q.data_ptr(), k.data_ptr(),
                       _dtype(out), ldq, ldk, _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return q, k


def _head_rows(fn, name, t, T, H, D, dtype, dev):
    """The row stride of an output given by the caller: [T, H * D] or [T, H, D], heads next to each other."""
    _check_rows(fn, name, t, None, dev)
    if (t.dtype != dtype or t.dim() not in (2, 3) or t.shape[0] != T
            or (t.shape[1] != H * D if t.dim() == 2 else tuple(t.shape[1:]) != (H, D) or (H > 1 and t.stride(1) != D))):
        _refuse(fn, f"{name} {tuple(t.shape)} {t.dtype}: [{T}, {H} * {D}] of {dtype}")
    ld = _stride_of(t.stride(0), H * D, T)
    if ld >> 31:
        _sizes(fn, ld)
    return ld


class GgufTensor:
    def __init__(self, name, qtype, dims, data, nbytes):
        self.name, self.qtype, self.dims, self.data, self.nbytes = name, qtype, dims, data, nbytes

    @property
    def K(self):
        return self.dims[0]

    @property
    def rows(self):
        r = 1
        for d in self.dims[1:]:
            r *= d
        return r

    def numpy(self):
        """The tensor's bytes as a uint8 numpy view of the mapping (valid while the file is open)."""
        import numpy as np
        return np.ctypeslib.as_array((ctypes.c_uint8 * self.nbytes).from_address(self.data))


class GgufFile:
    """A mapped GGUF file (qmatmul_gguf_*): tensors by name, metadata by key."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        _call("qmatmul_gguf_open", os.fsencode(path), ctypes.byref(h))
        self.handle = h

    def __len__(self):
        n = ctypes.c_int()
        _call("qmatmul_gguf_tensor_count", self.handle, ctypes.byref(n))
        return n.value

    def tensor(self, key):
        i = key
        if isinstance(key, str):
            idx = ctypes.c_int()
            _call("qmatmul_gguf_find_tensor", self.handle, key.encode(), ctypes.byref(idx))
            i = idx.value
        name, t, nd = ctypes.c_char_p(), ctypes.c_int(), ctypes.c_int()
        dims = (ctypes.c_uint64 * 8)()
        data, nb = ctypes.c_void_p(), ctypes.c_uint64()
        _call("qmatmul_gguf_tensor_info", self.handle, i, ctypes.byref(name), ctypes.byref(t), ctypes.byref(nd), dims,
              ctypes.byref(data), ctypes.byref(nb))
        return GgufTensor(name.value.decode(), t.value, [int(d) for d in dims[:nd.value]], data.value or 0, nb.value)

    def get_int(self, key):
        v = ctypes.c_int64()
        _call("qmatmul_gguf_get_int", self.handle, key.encode(), ctypes.byref(v))
        return v.value

    def get_float(self, key):
        v = ctypes.c_double()
        _call("qmatmul_gguf_get_float", self.handle, key.encode(), ctypes.byref(v))
        return v.value

    def get_str(self, key):
        v = ctypes.c_char_p()
        _call("qmatmul_gguf_get_str", self.handle, key.encode(), ctypes.byref(v))
        return v.value.decode()

    def close(self):
        if self.handle:
            _call("qmatmul_gguf_close", self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()
