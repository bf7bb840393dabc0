"""The paged cache's operators on their way from Python to the C ABI, without a GPU: tensors of the meta device stand for those of the
current GPU, the library's functions are recorded instead of called."""
import pytest
import torch

F32, F16, BF16, I32, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.float8_e4m3fn
FAR = 2 ** 32  # (modulo which ctypes takes an int)


@pytest.fixture()
def calls(qm, monkeypatch):
    """(function, arguments) of every call of the library."""
    made = []
    monkeypatch.setattr(qm, "_torch", torch)
    monkeypatch.setattr(qm, "_current_gpu", lambda: -1)  # (what get_device() says of a meta tensor)
    monkeypatch.setattr(qm, "_current_stream", lambda dev: 0)
    monkeypatch.setattr(qm, "_function", lambda name: lambda *a: made.append((name, a)) or 0)
    monkeypatch.setattr(qm, "_call", lambda name, *a: made.append((name, a)) or 0)
    return made


def meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def laid(shape, strides, dtype=BF16):
    return torch.empty_strided(shape, strides, dtype=dtype, device="meta")


def cache(qm, dtype=BF16, pages=8, heads=2, page=16, D=64, mean=True):
    scales = [meta(pages, heads, page, dtype=F32) for _ in range(2)] if dtype == E4M3 else [None, None]
    return qm.KvCache(meta(pages, heads, page, D, dtype=dtype), meta(pages, heads, page, D, dtype=dtype), *scales,
                      meta(pages, heads, D) if mean else None)


def attn(qm, T=3, B=3, kv=None, q=None, lens=None, table=None, **k):
    q = meta(T, 4, 64) if q is None else q
    return qm.attn_prefix(q, kv or cache(qm), meta(B, dtype=I32) if lens is None else lens, meta(B, 5, dtype=I32) if table is None else table, **k)


def chosen(qm, sel=None, **k):
    return qm.attn_pages(meta(3, 4, 64), cache(qm), meta(3, dtype=I32), meta(3, 5, dtype=I32), meta(3, 2, 4, dtype=I32) if sel is None else sel, **k)


def choice(qm, k=4, kv=None, W=4, **kw):
    return qm.select_pages(meta(3, 4, 64), kv or cache(qm), meta(3, dtype=I32), meta(3, W, dtype=I32), k, **kw)


def append(qm, x=None, HQ=4, kv=None, slots=None, pos=None, f=None, **k):
    return qm.kv_append(meta(3, 512) if x is None else x, HQ, kv or cache(qm), meta(3, dtype=I32) if slots is None else slots,
                        meta(3, dtype=I32) if pos is None else pos, meta(32, dtype=F32) if f is None else f, **k)


def test_these_calls_are_taken(qm, calls):
    assert attn(qm).dtype == BF16 and attn(qm, out=F32).dtype == F32
    attn(qm, T=7, start=meta(4, dtype=I32), prefix=meta(2, dtype=I32), prefix_len=20, scale=0.5)
    attn(qm, q=laid((3, 4, 64), (2 ** 31 - 1, 64, 1)), o=laid((3, 4, 64), (300, 64, 1)))
    attn(qm, kv=cache(qm, E4M3), q=meta(3, 4, 64, dtype=F16))
    chosen(qm)
    assert tuple(choice(qm).shape) == (3, 2, 4)
    assert append(qm).dtype == BF16 and append(qm, kv=cache(qm, E4M3)).dtype == BF16 and append(qm, kv=cache(qm, F16)).dtype == F16
    append(qm, x=meta(3, 256), HQ=0)
    qm.KvCache(laid((8, 2, 16, 64), (64, 8 * 16 * 64, 8 * 64, 1)), laid((8, 2, 16, 64), (64, 8 * 16 * 64, 8 * 64, 1)))
    names = [n for n, _ in calls]
    assert names.count("qmatmul_attn_prefix") == 5 and names.count("qmatmul_kv_append") == 4 and names[-5:-4] == ["qmatmul_select_pages"]
    assert calls[3][1][2] == 2 ** 31 - 1 and calls[3][1][-4] == 300 and calls[2][1][7:9] == (20, 0.5)


def test_caches(qm, calls):
    k = meta(8, 2, 16, 64)
    e, s = meta(8, 2, 16, 64, dtype=E4M3), meta(8, 2, 16, dtype=F32)
    for bad in (lambda: qm.KvCache(k, meta(8, 2, 16, 32)), lambda: qm.KvCache(k, meta(8, 2, 16, 64, dtype=F16)), lambda: qm.KvCache(meta(8, 2, 16, 64, dtype=F32), k),
                lambda: qm.KvCache(k, laid((8, 2, 16, 64), (64, 8 * 16 * 64, 8 * 64, 1))), lambda: qm.KvCache(k[0], k[0]), lambda: qm.KvCache(k, k, s, s),
                lambda: qm.KvCache(e, e), lambda: qm.KvCache(e, e, s), lambda: qm.KvCache(e, e, s, meta(8, 2, 15, dtype=F32)),
                lambda: qm.KvCache(e, e, s, meta(8, 2, 16, dtype=F16)), lambda: qm.KvCache(e, e, s, meta(8, 16, 2, dtype=F32).transpose(1, 2)),
                lambda: qm.KvCache(k, k, mean=meta(8, 2, 64, dtype=F32)), lambda: qm.KvCache(k, k, mean=meta(8, 64)),
                lambda: qm.KvCache(k.transpose(2, 3), k.transpose(2, 3)), lambda: qm.KvCache(meta(FAR + 8, 1, 16, 16), meta(FAR + 8, 1, 16, 16)),
                lambda: qm.KvCache(meta(8, 2, 32, 64)[:, :, ::2], k)):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls


def test_refused(qm, calls):
    i32 = lambda *n: meta(*n, dtype=I32)  # noqa: E731
    for bad in (lambda: attn(qm, q=meta(3, 4, 32)), lambda: attn(qm, q=meta(3, 256)), lambda: attn(qm, q=laid((3, 4, 64), (512, 128, 1))),
                lambda: attn(qm, q=laid((3, 4, 64), (256, 64, 2))), lambda: attn(qm, q=laid((3, 4, 64), (FAR + 256, 64, 1))),
                lambda: attn(qm, o=laid((3, 4, 64), (FAR + 256, 64, 1))), lambda: attn(qm, o=meta(2, 4, 64)), lambda: attn(qm, o=meta(3, 4, 64), out=F32),
                lambda: attn(qm, B=2), lambda: attn(qm, table=i32(2, 5)), lambda: attn(qm, table=i32(3, 10)[:, ::2]), lambda: attn(qm, table=meta(3, 5, dtype=F32)),
                lambda: attn(qm, table=i32(3, FAR + 5)), lambda: attn(qm, lens=meta(3, dtype=torch.int64)), lambda: attn(qm, start=i32(3)),
                lambda: attn(qm, start=meta(4, dtype=F32)), lambda: attn(qm, prefix_len=5), lambda: attn(qm, prefix=i32(1), prefix_len=17),
                lambda: attn(qm, prefix=i32(1), prefix_len=-1), lambda: attn(qm, prefix=i32(2 ** 30), prefix_len=FAR + 5),
                lambda: chosen(qm, sel=i32(3, 4, 4)), lambda: chosen(qm, sel=i32(2, 2, 4)), lambda: chosen(qm, sel=i32(3, 2, 8)[..., ::2]),
                lambda: chosen(qm, sel=meta(3, 2, 4, dtype=F32)), lambda: choice(qm, kv=cache(qm, mean=False)), lambda: choice(qm, k=FAR + 4),
                lambda: choice(qm, first=FAR + 1), lambda: choice(qm, sel=i32(3, 2, 5)), lambda: choice(qm, sel=i32(3, 4, 2).transpose(1, 2)),
                lambda: append(qm, slots=i32(2)), lambda: append(qm, slots=meta(3, dtype=torch.int64)), lambda: append(qm, slots=i32(6)[::2]),
                lambda: append(qm, pos=i32(2)), lambda: append(qm, pos=meta(3, dtype=F32)), lambda: append(qm, f=meta(32, dtype=F16)),
                lambda: append(qm, wq=meta(32, dtype=F32)), lambda: append(qm, wk=meta(64)), lambda: append(qm, x=meta(3, 511)), lambda: append(qm, HQ=-1),
                lambda: append(qm, HQ=FAR + 4, x=laid((3, 64 * (FAR + 8)), (2 ** 31 - 1, 1))), lambda: append(qm, v_off=449), lambda: append(qm, sections=(16, 15)),
                lambda: append(qm, x=laid((3, 512), (FAR + 512, 1))), lambda: append(qm, q=laid((3, 256), (FAR + 256, 1))), lambda: append(qm, q=meta(3, 4, 64), out=F32),
                lambda: qm.attn_workspace(cache(qm), FAR + 1, 1, 4), lambda: qm.select_workspace(cache(qm), 1, FAR)):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls


def test_tensors_without_dimensions_are_refused(qm, calls):
    none = lambda dtype=BF16: meta(dtype=dtype)  # noqa: E731
    for bad in (lambda: append(qm, pos=none(I32)), lambda: append(qm, x=none()), lambda: append(qm, slots=none(I32)), lambda: append(qm, f=none(F32)),
                lambda: append(qm, wq=none(F32)), lambda: append(qm, wk=none(F32)), lambda: append(qm, q=none()), lambda: attn(qm, q=none()), lambda: attn(qm, o=none()),
                lambda: attn(qm, lens=none(I32)), lambda: attn(qm, table=none(I32)), lambda: attn(qm, start=none(I32)), lambda: attn(qm, ws=none(torch.uint8)),
                lambda: attn(qm, prefix=none(I32), prefix_len=1), lambda: chosen(qm, sel=none(I32)), lambda: choice(qm, sel=none(I32)),
                lambda: qm.attn_pages(none(), cache(qm), meta(3, dtype=I32), meta(3, 5, dtype=I32), meta(3, 2, 4, dtype=I32)), lambda: qm.KvCache(none(), none())):
        with pytest.raises(qm.QMatmulError):
            bad()
    assert not calls
