"""Pages more than 2^32 bytes into a cache, for each kernel that reads it: few rows and many, chosen pages, 8-bit values and their scales; the same bits as from a small
cache that holds the same pages."""
import pytest
import torch

from tests import kv_plain as K

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("ct", [BF16, E4M3])
def test_far_pages(qm, dev, ct):
    D, page, HK = 128, 64, 2
    size = 1 if ct == E4M3 else 2
    pages = (2 ** 32 + 2 ** 28) // (page * D * HK * size)
    far = [pages - 1, pages // 2 + 5, 3, pages - 70]
    small = K.Cache(4, HK, page, D, ct, 15)
    raw = torch.uint8 if ct == E4M3 else ct
    big = []
    for t in small.data:
        b = torch.empty((pages, HK, page, D), dtype=raw, device=dev)
        b[far] = t.view(raw).to(dev)
        big.append(b.view(ct))
    scales = []
    for s in small.scales:
        if s is not None:
            b = torch.empty((pages, HK, page), device=dev)
            b[far] = s.to(dev)
            scales.append(b)
    kv, near = qm.KvCache(*big, *scales), small.on(qm, dev)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    ln, tables = i32([250]), (i32([far]), i32([[0, 1, 2, 3]]))
    sel = i32([[2, 0], [3, 1]])
    for rows in (1, 5, 100):
        q = torch.randn((rows, 8, D), generator=torch.Generator().manual_seed(rows)).to(BF16).to(dev)
        start = i32([0, rows])
        a, b = (qm.attn_prefix(q, c, ln, t, start=start) for c, t in ((kv, tables[0]), (near, tables[1])))
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())
        a, b = (qm.attn_prefix(q, c, i32([0]), t, start=start, prefix=t[0], prefix_len=250, ws=qm.attn_workspace(c, rows, 1, 8, 250))
                for c, t in ((kv, tables[0]), (near, tables[1])))
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())
        pick = sel.expand(rows, 2, 2).contiguous()
        a, b = (qm.attn_pages(q, c, ln, t, pick, start=start) for c, t in ((kv, tables[0]), (near, tables[1])))
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())


def test_far_means(qm, dev):
    """Means 2^32 bytes into their list."""
    D, HK = 256, 4
    pages = (2 ** 32 + 2 ** 26) // (HK * D * 2)
    k = torch.empty((1,), dtype=BF16, device=dev).expand(pages, HK, 16, D)  # (not read)
    mean = torch.zeros((pages, HK, D), dtype=BF16, device=dev)
    kv = qm.QmKv(30, D, HK, 16, pages, 0, 0, 0, k.data_ptr(), k.data_ptr(), None, None, mean.data_ptr())
    q = torch.randn((1, 8, D), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    far = list(range(pages - 40, pages))
    mean[far] = torch.randn((40, HK, D), generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    near = qm.KvCache(*[torch.zeros((40, HK, 16, D), dtype=BF16, device=dev) for _ in range(2)], mean=mean[far].contiguous())
    ln = torch.tensor([640], dtype=torch.int32, device=dev)
    want = qm.select_pages(q, near, ln, torch.arange(40, dtype=torch.int32, device=dev)[None], 7)
    cache = qm.KvCache.__new__(qm.KvCache)
    import ctypes
    cache.view, cache.mean, cache.pages, cache.heads, cache.page, cache.D, cache.device_index = kv, mean, pages, HK, 16, D, near.device_index
    cache.ref = ctypes.byref(kv)
    got = qm.select_pages(q, cache, ln, torch.tensor([far], dtype=torch.int32, device=dev), 7)
    assert torch.equal(got, want)


def test_far_rows(qm, dev):
    """Rows of q, of the result and of the QKV product more than 2^31 elements behind the first one."""
    T, HQ, HK, D, far = 4, 8, 2, 64, 2 ** 30
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    buf = torch.empty(((T - 1) * far + (HQ + 2 * HK) * D,), dtype=BF16, device=dev)
    x = torch.randn((T, (HQ + 2 * HK) * D), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    rows = buf.as_strided(x.shape, (far, 1))
    rows.copy_(x)
    near, kv = (qm.KvCache.new(2, HK, 16, D, BF16) for _ in range(2))
    pos, f = i32([3, 4, 5, 6]), torch.rand(D // 2, generator=torch.Generator().manual_seed(2)).to(dev)
    q = qm.kv_append(x, HQ, near, pos, pos, f)
    got = qm.kv_append(rows, HQ, kv, pos, pos, f, q=rows[:, :HQ * D])  # (in place)
    assert torch.equal(got, q.view(T, HQ * D)) and torch.equal(kv.k, near.k) and torch.equal(kv.v, near.v)
    q4 = buf.as_strided((T, HQ, D), (far, D, 1))
    out = torch.empty(((T - 1) * far + HQ * D,), dtype=BF16, device=dev)
    o = out.as_strided((T, HQ, D), (far, D, 1))
    for start, ln, table in ((None, i32([4, 5, 6, 7]), i32([[0]] * 4)), (i32([0, 4]), i32([7]), i32([[0]]))):
        want = qm.attn_prefix(q, kv, ln, table, start=start)
        qm.attn_prefix(q4, kv, ln, table, start=start, o=o)
        assert torch.equal(o, want)
        out.zero_()
        qm.attn_pages(q4, kv, ln, table, i32([0]).expand(T, HK, 1).contiguous(), start=start, o=o)
        assert torch.equal(o, qm.attn_pages(q, kv, ln, table, i32([0]).expand(T, HK, 1).contiguous(), start=start))


def test_far_rows_of_large_tiles(qm, dev):
    """The same for a prompt: 70 rows, the last of them more than 2^31 elements behind the first."""
    T, HQ, HK, D, far = 70, 2, 1, 128, 2 ** 25
    cache = K.Cache(8, HK, 16, D, BF16, 5)
    kv, ln, table = cache.on(qm, dev), torch.tensor([100], dtype=torch.int32, device=dev), torch.arange(8, dtype=torch.int32, device=dev)[None]
    start = torch.tensor([0, T], dtype=torch.int32, device=dev)
    q = torch.randn((T, HQ, D), generator=torch.Generator().manual_seed(6)).to(BF16).to(dev)
    bufs = [torch.empty(((T - 1) * far + HQ * D,), dtype=BF16, device=dev) for _ in range(2)]
    rows, o = (b.as_strided((T, HQ, D), (far, D, 1)) for b in bufs)
    rows.copy_(q)
    qm.attn_prefix(rows, kv, ln, table, start=start, o=o)
    assert torch.equal(o, qm.attn_prefix(q, kv, ln, table, start=start))
