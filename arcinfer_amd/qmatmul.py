"""ctypes binding of libqmatmul.so (include/qmatmul.h) and torch-tensor conveniences.

The library is the product: this module only passes device pointers and sizes through the C ABI. It raises
QMatmulError for any non-zero status, and refuses to run when the library is not built (there is no fallback).

Calls run on torch's current stream, or on `stream`, the raw handle of another one. Inputs have to be ready there; results that the caller does not
give are made there too, as under torch.cuda.stream.
"""
import ctypes
import functools
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
    ("qmatmul_kv_append", _I, [_P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _c.c_float, _P, _P, _I, _P, _P, _P, _P, _I, _I, _P]),
    ("qmatmul_attn_workspace_size", _Z, [_P, _I, _I, _I, _I]),
    ("qmatmul_attn_prefix", _I, [_P, _I, _I, _I, _P, _P, _P, _I, _c.c_float, _P, _I, _I, _P, _Z, _P]),
    ("qmatmul_select_workspace_size", _Z, [_P, _I, _I]),
    ("qmatmul_select_pages", _I, [_P, _I, _I, _I, _P, _P, _I, _I, _I, _P, _P, _Z, _P]),
    ("qmatmul_attn_pages", _I, [_P, _I, _I, _I, _P, _P, _P, _I, _c.c_float, _P, _I, _I, _P, _Z, _P]),
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


def _on(stream, dev, make):
    """What makes a call's results, and a workspace that it keeps to itself, where the caller names a stream: `make` with that stream as the current one. A fill
    then comes before the kernel, the memory is none that the current stream still works on, and nobody else gets it before that stream is done with it."""
    if stream is None:
        return make
    stream = getattr(stream, "value", stream) or 0  # (of a ctypes pointer)
    if stream == _current_stream(dev):
        return make
    import torch

    def made(*args, **more):
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev)):
            return make(*args, **more)
    return made


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
    aq, asc, absum = _on(stream, x.device.index, _out_acts)(Ms, K, x.device, act32)
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
        C = _on(stream, aq.device.index, torch.empty)((T, w.rows), dtype=torch.float32, device=aq.device)
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
        C = _on(stream, aq.device.index, torch.empty)((M, w.rows), dtype=torch.float32, device=aq.device)
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
        C = _on(stream, aq.device.index, torch.empty)((M, w.rows), dtype=torch.float32, device=aq.device)
        ldc = w.rows
    _call("qmatmul_gemm_ws", w.handle, _ptr(aq), _ptr(asc), _ptr(absum), M, Ms, int(act32), _ptr(C),
          w.rows if ldc is None else ldc, c_off, accumulate, _ptr(ws), 0 if ws is None else ws.numel(),
          _stream(stream))
    return C


def gemv_blocksums(w, aq, absum, T=1, stream=None):
    import torch
    nb = w.K // 32
    empty = _on(stream, aq.device.index, torch.empty)
    isum = empty((T, w.rows, nb), dtype=torch.int32, device=aq.device)
    msum = empty((T, w.rows, nb), dtype=torch.int32, device=aq.device) if w.qtype in (12, 13, 10) else None
    _call("qmatmul_gemv_blocksums", w.handle, _ptr(aq), _ptr(absum), aq.shape[0], T, _ptr(isum), _ptr(msum),
          _stream(stream))
    return isum, msum


def gemm_blocksums(w, aq, M=None, stream=None):
    import torch
    M = aq.shape[0] if M is None else M
    isum = _on(stream, aq.device.index, torch.empty)((M, w.rows, w.K // 32), dtype=torch.int32, device=aq.device)
    _call("qmatmul_gemm_blocksums", w.handle, _ptr(aq), M, aq.shape[0], _ptr(isum), _stream(stream))
    return isum


def moe_route(logits, NU, NE=None, stream=None):
    import torch
    T, ldl = logits.shape
    NE = ldl if NE is None else NE
    empty = _on(stream, logits.device.index, torch.empty)
    ids = empty((T, NU), dtype=torch.int32, device=logits.device)
    wts = empty((T, NU), dtype=torch.float32, device=logits.device)
    counts = empty((NE,), dtype=torch.int32, device=logits.device)
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
    aq, asc, absum = _on(stream, x.device.index, _out_acts)(Ms, K, x.device, act32)
    h = _on(stream, x.device.index, torch.empty)((Ms, K), dtype=torch.float32, device=x.device) if want_h else None
    _call("qmatmul_rmsnorm_quant_ex", _ptr(x), x.stride(0), _ptr(w), K, M, Ms, float(eps), int(act32), _ptr(aq),
          _ptr(asc), _ptr(absum), _ptr(h), K, _stream(stream))
    return aq, asc, absum, h


def swiglu_quant(gu, F, fused=False, gelu=False, M_stride=None, stream=None, act32=True):
    M = gu.shape[0]
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _on(stream, gu.device.index, _out_acts)(Ms, F, gu.device, act32)
    _call("qmatmul_swiglu_quant_ex", _ptr(gu), gu.stride(0), F, M, Ms, int(fused), int(gelu), int(act32), _ptr(aq),
          _ptr(asc), _ptr(absum), _stream(stream))
    return aq, asc, absum


def add_norm_quant(x, t, w, eps, s, w2=None, M_stride=None, stream=None, act32=True):
    """Updates x in place; returns (aq, asc, absum)."""
    M, K = x.shape
    Ms = M if M_stride is None else M_stride
    aq, asc, absum = _on(stream, x.device.index, _out_acts)(Ms, K, x.device, act32)
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
    """t is on GPU `dev`, of `dim` dimensions where dim is given (one at least where it is not), its last one contiguous."""
    if t.get_device() == dev and (t.dim() == dim if dim else t.dim()) and t.stride(-1) == 1:
        return
    if t.get_device() != dev:
        _refuse(fn, f"{name} is on {t.device}, not on the current GPU")
    if t.dim() != dim if dim else not t.dim():
        _refuse(fn, f"{name} has {t.dim()} dimensions, not {dim or 'one or more'}")
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


def _out_fp8(fn, x, M, K, M_stride, stream, dev):
    """(M_stride, ldx, a8, asc) of a producer's rows x; where M_stride is 0 there is nothing to call for."""
    Ms, ldx = M if M_stride is None else M_stride, x.stride(0) if M > 1 else _row_stride(x)
    if (M | Ms | K | ldx) >> 31 or Ms == 0:
        _sizes(fn, M, Ms, K, ldx)
        _dtype(x.dtype)
        if Ms < M or K < 1:
            _refuse(fn, f"M {M}, M_stride {Ms}, K {K}")
    Kp = (K + 127) // 128 * 128
    empty = x.new_empty if stream is None else _on(stream, dev, x.new_empty)  # (the test here: a call that names none pays nothing)
    return Ms, ldx, empty((Ms, Kp), dtype=_torch.float8_e4m3fn), empty((Kp // 128, Ms), dtype=_torch.float32)


def quantize_fp8(x, M_stride=None, stream=None):
    """x [M, K] (float32, float16 or bfloat16, rows of any stride) -> (a8 float8_e4m3fn [M_stride, Kp], asc float32
    [Kp / 128, M_stride]), Kp = K rounded up to 128."""
    fn = "qmatmul_quantize_fp8"
    dev = _current_gpu()
    _check_rows(fn, "x", x, 2, dev)
    M, K = x.shape
    Ms, ldx, a8, asc = _out_fp8(fn, x, M, K, M_stride, stream, dev)
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
    Ms, ldx, a8, asc = _out_fp8(fn, x, M, K, M_stride, stream, dev)
    h = _on(stream, dev, x.new_empty)((M, K), dtype=torch.float32) if want_h else None
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
    Ms, ldg, a8, asc = _out_fp8(fn, gu, M, F, M_stride, stream, dev)
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
        C = (asc.new_empty if stream is None else _on(stream, dev, asc.new_empty))((M, w.rows), dtype=out)
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
    empty = x.new_empty if stream is None else _on(stream, dev, x.new_empty)
    if q is None:
        q, ldq = empty((T, HQ, D), dtype=out), HQ * D
    else:
        ldq = _head_rows(fn, "q", q, T, HQ, D, out, dev)
    if k is None:
        k, ldk = empty((T, HK, D), dtype=out), HK * D
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


# ---- keys and values in pages, and attention over them ----------------------------------------------------------------
class QmKv(ctypes.Structure):
    _fields_ = [("type", _I), ("D", _I), ("heads", _I), ("page", _I), ("pages", _I), ("page_stride", _c.c_longlong),
                ("head_stride", _c.c_longlong), ("token_stride", _c.c_longlong), ("k", _P), ("v", _P), ("k_scale", _P),
                ("v_scale", _P), ("mean", _P)]


class QmSeqs(ctypes.Structure):
    _fields_ = [("T", _I), ("B", _I), ("start", _P), ("len", _P), ("table", _P), ("table_stride", _I)]


class KvCache:
    """One layer's keys and values in pages: k, v [pages, heads, page, D] of float16, bfloat16 or float8_e4m3fn (views of any order
    in memory, both of one; the last dimension contiguous), with k_scale, v_scale float32 [pages, heads, page] for 8 bits, and
    mean bfloat16 [pages, heads, D] where pages are to be selected. The tensors stay the caller's."""

    def __init__(self, k, v, k_scale=None, v_scale=None, mean=None):
        import torch
        fn = "KvCache"
        dev = _current_gpu()
        kinds = {torch.float16: 1, torch.bfloat16: 30, torch.float8_e4m3fn: 256}
        for name, t in (("k", k), ("v", v)):
            _check_rows(fn, name, t, 4, dev)
            if t.dtype not in kinds:
                raise QMatmulError(fn, 3, f"{name} of {t.dtype}: float16, bfloat16 or float8_e4m3fn")
        if k.shape != v.shape or k.dtype != v.dtype or any(a != b for a, b, n in zip(k.stride(), v.stride(), k.shape) if n > 1):
            _refuse(fn, f"k {tuple(k.shape)} {k.dtype} {k.stride()} and v {tuple(v.shape)} {v.dtype} {v.stride()} are laid out differently")
        pages, heads, page, D = k.shape
        _sizes(fn, pages, heads, page, D)
        if (k_scale is None) != (k.dtype != torch.float8_e4m3fn) or (k_scale is None) != (v_scale is None):
            _refuse(fn, "k_scale and v_scale belong to float8_e4m3fn, and to nothing else")
        for name, t, shape, dtype in (("k_scale", k_scale, (pages, heads, page), torch.float32), ("v_scale", v_scale, (pages, heads, page), torch.float32),
                                      ("mean", mean, (pages, heads, D), torch.bfloat16)):
            if t is not None:
                _check_rows(fn, name, t, 3, dev)
                if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
                    _refuse(fn, f"{name} {tuple(t.shape)} {t.dtype}: contiguous {dtype} {shape}")
        self.k, self.v, self.k_scale, self.v_scale, self.mean = k, v, k_scale, v_scale, mean
        self.pages, self.heads, self.page, self.D, self.dtype, self.device_index = pages, heads, page, D, k.dtype, dev
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.view = QmKv(kinds[k.dtype], D, heads, page, pages, k.stride(0), k.stride(1), k.stride(2), k.data_ptr(), v.data_ptr(),
                         at(k_scale), at(v_scale), at(mean))
        self.ref = ctypes.byref(self.view)

    @classmethod
    def new(cls, pages, heads, page, D, dtype, mean=False):
        """An empty cache on the current GPU."""
        import torch
        made = lambda *shape, dtype: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        k, v = (made(pages, heads, page, D, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype) for _ in range(2))
        scales = [made(pages, heads, page, dtype=torch.float32) for _ in range(2)] if dtype == torch.float8_e4m3fn else [None, None]
        return cls(k.view(dtype), v.view(dtype), *scales, made(pages, heads, D, dtype=torch.bfloat16) if mean else None)


def _check_int32(fn, name, t, dim, dev):
    _check_rows(fn, name, t, dim, dev)
    if t.dtype != _torch.int32 or not t.is_contiguous():
        _refuse(fn, f"{name} {tuple(t.shape)} {t.dtype}: contiguous int32")


def _check_cache(fn, kv, dev):
    if kv.device_index != dev:
        _refuse(fn, "the cache is not on the current GPU")


_rotations = {}  # QmRope by what it says


def kv_append(x, HQ, kv, slots, pos, inv_freq, wq=None, wk=None, eps=1e-6, adjacent=False, sections=None, turns=False, scale=1.0,
              q_off=0, q_hs=None, k_off=None, k_hs=None, v_off=None, v_hs=None, q=None, out=None, stream=None):
    """qk_norm_rope of rows x [T, ldx] with the keys and the value heads (neither normed nor turned) to a KvCache: token t to its place
    slots[t] (int32 [T]: page * tokens of a page + place in it; one outside the cache, as a negative one, is not stored; no two the same).
    Value head h is at column v_off + h * v_hs (behind the key heads unless given). With kv.mean: the mean key of each page whose last
    token is among these. Returns q [T, HQ, D] of type out (that of a given q, else the cache's, bfloat16 for an 8-bit one), or the q given."""
    # (Appending a few tokens takes the GPU 5 us: each check is made in the cheapest way, and only what fails it goes to the functions that say why.)
    fn = "qmatmul_kv_append"
    dev = _current_gpu()
    torch = _torch
    D, HK = kv.D, kv.heads
    if kv.device_index != dev:
        _check_cache(fn, kv, dev)
    sx, sp, one = x.stride(), pos.stride(), (1,)
    if x.get_device() != dev or len(sx) != 2 or sx[1] != 1:
        _check_rows(fn, "x", x, 2, dev)
    T, width = x.shape
    if slots.get_device() != dev or slots.dtype != torch.int32 or slots.stride() != one:
        _check_int32(fn, "slots", slots, 1, dev)
    axes, half = 1, inv_freq.numel()
    if len(sp) > 1:
        axes = pos.size(0)
    if pos.get_device() != dev or sp[-1:] != one:
        _check_rows(fn, "pos", pos, None, dev)
    if inv_freq.get_device() != dev or inv_freq.stride() != one:
        _check_rows(fn, "inv_freq", inv_freq, 1, dev)
    if pos.dtype != torch.int32 or len(sp) > 2 or pos.shape[-1] != T or slots.numel() != T:
        _refuse(fn, f"pos {tuple(pos.shape)} {pos.dtype}, slots {tuple(slots.shape)}: int32, one column for each of {T} tokens")
    f32 = torch.float32
    if inv_freq.dtype != f32:
        _refuse(fn, f"inv_freq {inv_freq.dtype}: float32")
    for w in (wq, wk):
        if w is not None:
            if w.get_device() != dev or w.stride() != one:
                _check_rows(fn, "wq or wk", w, 1, dev)
            if w.dtype != f32 or w.numel() != D:
                _refuse(fn, f"wq or wk {tuple(w.shape)} {w.dtype}: float32 [{D}]")
    if sections is None:
        sections = (half,)
    if len(sections) != axes or axes > 4 or sum(sections) != half:
        _refuse(fn, f"sections {sections}: one for each of {axes} axes (at most 4), their sum {half}")
    if q_hs is None:
        q_hs = D
    if k_hs is None:
        k_hs = D
    if v_hs is None:
        v_hs = D
    if k_off is None:
        k_off = q_off + HQ * q_hs
    if v_off is None:
        v_off = k_off + HK * k_hs
    ldx, ps = sx[0] if T > 1 else _row_stride(x), sp[0] if axes > 1 else T
    if (T | HQ | ldx | ps | q_off | q_hs | k_off | k_hs | v_off | v_hs | 2 * half) >> 31 or (axes > 1 and min(sections) < 0):
        _sizes(fn, T, HQ, ldx, ps, q_off, q_hs, k_off, k_hs, v_off, v_hs, 2 * half, *sections)
        if HQ < 0:
            _refuse(fn, f"HQ {HQ}")
    if max(q_off + (HQ - 1) * q_hs if HQ else 0, k_off + (HK - 1) * k_hs, v_off + (HK - 1) * v_hs) + D > width:
        _refuse(fn, f"rows of {width} elements do not hold the heads")
    if out is None:
        out = q.dtype if q is not None else kv.dtype if kv.dtype != torch.float8_e4m3fn else torch.bfloat16
    if q is None:
        q, ldq = (x.new_empty if stream is None else _on(stream, dev, x.new_empty))((T, HQ, D), dtype=out), HQ * D
    else:
        ldq = _head_rows(fn, "q", q, T, HQ, D, out, dev)
    how = (2 * half, adjacent, turns, scale, *sections)
    rope = _rotations.get(how)
    if rope is None:
        if len(_rotations) >= 64:
            _rotations.clear()
        rope = _rotations[how] = ctypes.pointer(QmRope(2 * half, adjacent, axes, turns, tuple(sections), scale))
    st = _function(fn)(x.data_ptr(), _dtype(x.dtype), ldx, T, q_off, q_hs, HQ, k_off, k_hs, v_off, v_hs,
                       None if wq is None else wq.data_ptr(), None if wk is None else wk.data_ptr(), eps, rope,
                       pos.data_ptr(), ps, inv_freq.data_ptr(), slots.data_ptr(), kv.ref, q.data_ptr(), _dtype(out), ldq,
                       _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return q


def _query(fn, q, kv, dev):
    """(T, HQ, ldq) of queries [T, HQ, D] (heads next to each other)."""
    _check_cache(fn, kv, dev)
    _check_rows(fn, "q", q, 3, dev)
    T, HQ, D = q.shape
    if D != kv.D or (HQ > 1 and q.stride(1) != D):
        _refuse(fn, f"q {tuple(q.shape)}, strides {q.stride()}: heads of {kv.D} next to each other")
    ldq = _stride_of(q.stride(0), HQ * D, T)
    if (T | HQ | ldq) >> 31:
        _sizes(fn, T, HQ, ldq)
    return T, HQ, ldq


def _batch(fn, T, lens, table, start, dev):
    _check_int32(fn, "lens", lens, 1, dev)
    _check_int32(fn, "table", table, 2, dev)
    B = lens.numel()
    if start is not None:
        _check_int32(fn, "start", start, 1, dev)
    if table.size(0) != B or (T != B if start is None else start.numel() != B + 1):
        _refuse(fn, f"{T} rows, lens {tuple(lens.shape)}, table {tuple(table.shape)}, start {None if start is None else tuple(start.shape)}: "
                    "a length and a row of pages for each sequence, start one more (or a row of q for each)")
    _sizes(fn, B, table.size(1))
    return QmSeqs(T, B, None if start is None else start.data_ptr(), lens.data_ptr(), table.data_ptr(), table.size(1))


def _workspace(fn, ws, dev):
    if ws is None:
        return None, 0
    _check_rows(fn, "ws", ws, 1, dev)
    return ws.data_ptr(), ws.numel() * ws.element_size()


def attn_workspace(kv, T, B, HQ, prefix_len=0):
    """A workspace for attn_prefix of T rows of B sequences (None where it needs none), or with B = T for attn_pages. Its size grows
    with neither the lengths nor the cache."""
    import torch
    fn = "qmatmul_attn_workspace_size"
    _sizes(fn, T, B, HQ, prefix_len)
    n = _function(fn)(kv.ref, T, B, HQ, prefix_len)
    return torch.empty((n,), dtype=torch.uint8, device="cuda") if n else None


def _attention(fn, q, kv, lens, table, start, scale, o, out, ws, stream, *more):
    dev = _current_gpu()
    T, HQ, ldq = _query(fn, q, kv, dev)
    seqs = _batch(fn, T, lens, table, start, dev)
    if out is None:
        out = q.dtype if o is None else o.dtype
    if o is None:
        # (rows of no sequence are not written: without a list of rows there are none)
        make = q.new_empty if start is None else q.new_zeros
        o, ldo = (make if stream is None else _on(stream, dev, make))((T, HQ, kv.D), dtype=out), HQ * kv.D
    else:
        ldo = _head_rows(fn, "o", o, T, HQ, kv.D, out, dev)
    ws_ptr, ws_bytes = _workspace(fn, ws, dev)
    st = _function(fn)(q.data_ptr(), _dtype(q.dtype), ldq, HQ, ctypes.byref(seqs), kv.ref, *more, kv.D ** -0.5 if scale is None else scale,
                       o.data_ptr(), _dtype(out), ldo, ws_ptr, ws_bytes, _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return o


def attn_prefix(q, kv, lens, table, start=None, prefix=None, prefix_len=0, scale=None, o=None, out=None, ws=None, stream=None):
    """Attention of q [T, HQ, D] (float16 or bfloat16, the cache's type unless that is of 8 bits) over a KvCache: over prefix_len tokens that
    all sequences share, in pages prefix (int32), and over each sequence's own up to the row itself. Sequence b has lens[b] tokens (int32
    [B]), these rows among them, in pages table[b] (int32 [B, pages]), and rows start[b] .. start[b + 1] - 1 of q (int32 [B + 1]; None: row b).
    scale: D ** -0.5 unless given. Returns o [T, HQ, D] of type out (q's, or float32; rows of no sequence zeros), or writes the o given (rows of no
    sequence stay). ws: of attn_workspace, for one call at a time; without one the prefix is not shared and long sequences not cut."""
    fn = "qmatmul_attn_prefix"
    prefix_ptr = None
    if prefix_len:
        _sizes(fn, prefix_len)
        if prefix is None:
            _refuse(fn, "prefix_len without a prefix")
        _check_int32(fn, "prefix", prefix, 1, _current_gpu())
        if prefix_len < 0 or prefix.numel() * kv.page < prefix_len:
            _refuse(fn, f"{prefix.numel()} pages of {kv.page} tokens do not hold a prefix of {prefix_len}")
        prefix_ptr = prefix.data_ptr()
    return _attention(fn, q, kv, lens, table, start, scale, o, out, ws, stream, prefix_ptr, prefix_len)


def attn_pages(q, kv, lens, table, sel, start=None, scale=None, o=None, out=None, ws=None, stream=None):
    """attn_prefix (without a prefix) over chosen pages only: sel int32 [T, heads, k], numbers of pages in the row's sequence for each key
    head, others than those of the table none (-1). ws: of attn_workspace(kv, T, T, HQ)."""
    fn = "qmatmul_attn_pages"
    _check_int32(fn, "sel", sel, 3, _current_gpu())
    if tuple(sel.shape[:2]) != (*q.shape[:1], kv.heads):
        _refuse(fn, f"sel {tuple(sel.shape)}, q {tuple(q.shape)}: pages for each row and each of {kv.heads} key heads")
    _sizes(fn, sel.size(2))
    return _attention(fn, q, kv, lens, table, start, scale, o, out, ws, stream, sel.data_ptr(), sel.size(2))


def select_workspace(kv, T, pages):
    """A workspace for select_pages of T rows with tables of `pages` pages."""
    import torch
    fn = "qmatmul_select_workspace_size"
    _sizes(fn, T, pages)
    n = _function(fn)(kv.ref, T, pages)
    return torch.empty((n,), dtype=torch.uint8, device="cuda") if n else None


def select_pages(q, kv, lens, table, k, start=None, first=1, last=1, sel=None, ws=None, stream=None):
    """The k pages of its sequence that each row's query heads score highest, by the pages' mean keys (kv.mean), the `first` first and `last`
    last ones always among them: int32 [T, heads, k], ascending, -1 behind them, for attn_pages (rows of no sequence: -1; in a sel
    given they stay). ws: of select_workspace; made for the call where it is not given and needed."""
    fn = "qmatmul_select_pages"
    dev = _current_gpu()
    T, HQ, ldq = _query(fn, q, kv, dev)
    seqs = _batch(fn, T, lens, table, start, dev)
    if kv.mean is None:
        _refuse(fn, "the cache has no means")
    _sizes(fn, k, first, last)
    if sel is None:
        make = lens.new_empty if start is None else functools.partial(lens.new_full, fill_value=-1)
        sel = (make if stream is None else _on(stream, dev, make))((T, kv.heads, k))
    else:
        _check_int32(fn, "sel", sel, 3, dev)
        if tuple(sel.shape) != (T, kv.heads, k):
            _refuse(fn, f"sel {tuple(sel.shape)}: [{T}, {kv.heads}, {k}]")
    if ws is None and table.size(1) > k:
        ws = _on(stream, dev, select_workspace)(kv, T, table.size(1))
    ws_ptr, ws_bytes = _workspace(fn, ws, dev)
    st = _function(fn)(q.data_ptr(), _dtype(q.dtype), ldq, HQ, ctypes.byref(seqs), kv.ref, k, first, last, sel.data_ptr(), ws_ptr, ws_bytes,
                       _current_stream(dev) if stream is None else stream)
    _done(fn, st)
    return sel


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
