"""Calls that name a stream: what they make for themselves and for the caller is made on it (allocations and fills), not on torch's current one. Without a GPU:
tensors of the meta device, streams that are recorded."""
import contextlib
import ctypes
from types import SimpleNamespace

import pytest
import torch

F32, F16, BF16, I32, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.float8_e4m3fn


@pytest.fixture()
def made(qm, monkeypatch):
    """Which streams are current at the allocations of a call (0: torch's current one)."""
    at, seen = [0], []
    monkeypatch.setattr(qm, "_torch", torch)
    monkeypatch.setattr(qm, "_current_gpu", lambda: -1)  # (what get_device() says of a meta tensor)
    monkeypatch.setattr(qm, "_current_stream", lambda dev: at[-1])
    monkeypatch.setattr(qm, "_function", lambda name: lambda *a: 512 if name.endswith("_size") else 0)
    monkeypatch.setattr(qm, "_call", lambda name, *a: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)

    @contextlib.contextmanager
    def current(s):
        at.append(s)
        yield
        at.pop()
    monkeypatch.setattr(torch.cuda, "stream", current)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: handle)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
    for name in ("new_empty", "new_zeros", "new_full"):
        real = getattr(torch.Tensor, name)
        monkeypatch.setattr(torch.Tensor, name, lambda t, *a, real=real, **k: seen.append(at[-1]) or real(t, *a, **k))
    empty = torch.empty

    def on_meta(*a, **k):
        seen.append(at[-1])
        return empty(*a, **{**k, "device": "meta"})
    monkeypatch.setattr(torch, "empty", on_meta)

    def run(call, *a, **k):
        seen.clear()
        call(*a, **k)
        return set(seen)
    return SimpleNamespace(run=run, current=current)


def meta(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype, device="meta")


def cached(qm):
    kv = qm.KvCache(meta(8, 2, 16, 64), meta(8, 2, 16, 64), mean=meta(8, 2, 64))
    q, lens, table, start = meta(5, 4, 64), meta(3, dtype=I32), meta(3, 6, dtype=I32), meta(4, dtype=I32)
    return [(qm.kv_append, (meta(5, 512), 4, kv, meta(5, dtype=I32), meta(5, dtype=I32), meta(32, dtype=F32)), {}),
            (qm.attn_prefix, (q, kv, lens, table), dict(start=start)),
            (qm.attn_prefix, (q[:3], kv, lens, table), {}),
            (qm.attn_pages, (q, kv, lens, table, meta(5, 2, 4, dtype=I32)), dict(start=start)),
            (qm.select_pages, (q, kv, lens, table, 4), dict(start=start)),
            (qm.select_pages, (q[:3], kv, lens, table, 4), {})]


def check(made, calls):
    for f, args, more in calls:
        assert made.run(f, *args, **more) == {0}, f
        assert made.run(f, *args, **more, stream=7) == {7}, f
        with made.current(7):
            assert made.run(f, *args, **more) == {7}, f
            assert made.run(f, *args, **more, stream=7) == {7}, f
            assert made.run(f, *args, **more, stream=0) == {"default"}, f


def test_the_paged_cache(qm, made):
    check(made, cached(qm))


def test_the_other_calls(qm, made):
    """Producers, products, routing, the rotation."""
    weight = SimpleNamespace(handle=1, rows=256, qtype=12, K=256, Kp=256)
    x, w, acts = meta(5, 256, dtype=F32), meta(256, dtype=F32), (meta(5, 256, dtype=torch.int8), meta(8, 5, dtype=F32), meta(16, 5, dtype=torch.int16))
    check(made, [(qm.quantize_act, (x,), {}), (qm.quantize_act, (x,), dict(act32=False)), (qm.gemv, (weight, *acts), {}), (qm.gemm, (weight, *acts), {}),
                 (qm.gemm_ws, (weight, *acts, None), {}), (qm.gemv_blocksums, (weight, acts[0], acts[2]), {}), (qm.gemm_blocksums, (weight, acts[0]), {}),
                 (qm.moe_route, (meta(5, 8, dtype=F32), 2), {}), (qm.rmsnorm_quant, (x, w, 1e-6), dict(want_h=True)), (qm.swiglu_quant, (meta(5, 512, dtype=F32), 256), {}),
                 (qm.add_norm_quant, (x, x, w, 1e-6, 1.0), {}), (qm.quantize_fp8, (x,), {}), (qm.rmsnorm_fp8, (x, w, 1e-6), dict(want_h=True)),
                 (qm.swiglu_fp8, (meta(5, 512, dtype=F32), 256), {}), (qm.gemm_fp8, (weight, meta(5, 256, dtype=E4M3), meta(2, 5, dtype=F32)), dict(out=BF16)),
                 (qm.qk_norm_rope, (meta(5, 512), 4, 2, 64, meta(5, dtype=I32), meta(32, dtype=F32)), {})])


def test_a_pointer_serves_as_a_number(qm, made):
    for f, args, more in cached(qm) + [(qm.quantize_fp8, (meta(5, 256, dtype=F32),), {})]:
        assert made.run(f, *args, **more, stream=ctypes.c_void_p(7)) == {7}, f
        with made.current(7):
            assert made.run(f, *args, **more, stream=ctypes.c_void_p(None)) == {"default"}, f
