"""Attention over a paged cache on the GPU against its 64-bit form (tests/kv_plain.py)."""
import math

import pytest
import torch

from tests import kv_plain as K

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
KINDS = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]  # q, cache


def queries(T, HQ, D, dtype, seed):
    return (torch.randn((T, HQ, D), generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype)


def run(qm, dev, lens, new, HQ, HK, D, page, qt, ct, out=None, prefix_len=0, ws=True, seed=0, pages=None, order=(0, 1, 2), pad=0, scale=None):
    shared = (prefix_len + page - 1) // page
    need = sum((n + page - 1) // page for n in lens) + shared + 2
    cache = K.Cache(pages or need, HK, page, D, ct, seed)
    start, ln, table, rest = K.batch(lens, new, page, need, seed)
    prefix = torch.tensor(rest[:shared], dtype=torch.int32)
    T = int(start[-1])
    q = queries(T, HQ, D, qt, seed + 1)
    out = out or qt
    kv = cache.on(qm, dev, order, pad)
    one = all(n == 1 for n in new)
    w = qm.attn_workspace(kv, T, len(lens), HQ, prefix_len) if ws else None
    got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=None if one else start.to(dev),
                         prefix=prefix.to(dev) if shared else None, prefix_len=prefix_len, out=out, ws=w, scale=scale)
    assert got.shape == (T, HQ, D) and got.dtype == out
    K.check(got, *K.attention(q, cache, start, ln, table, out, scale, prefix, prefix_len), out)


@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D,page", [(16, 16), (64, 64), (80, 32), (96, 16), (128, 64), (144, 128), (192, 16), (256, 256)])
def test_decode(qm, dev, D, page, qt, ct):
    """One token a sequence: lengths of one, of whole blocks and beside them, over several pages."""
    run(qm, dev, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300], [1] * 12, 4, 2, D, page, qt, ct, seed=D)


@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("G", [1, 3, 5, 16, 17, 40])
def test_heads(qm, dev, G, qt, ct):
    run(qm, dev, [70, 5], [1, 1], 2 * G, 2, 64, 16, qt, ct, seed=G)
    run(qm, dev, [70, 45], [7, 2], G, 1, 128, 16, qt, ct, seed=G, ws=False)


@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_several_tokens(qm, dev, D, qt, ct, out):
    """New tokens of every count, a sequence of new tokens alone among them; row tiles that end inside a token's heads."""
    run(qm, dev, [1, 9, 40, 200, 66], [1, 9, 3, 33, 1], 6, 2, D, 16, qt, ct, out=out, seed=D)
    run(qm, dev, [130, 90], [130, 50], 2, 2, D, 32, qt, ct, out=out, seed=D + 1)


@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("prefix_len", [1, 31, 100, 256, 300, 1000])
@pytest.mark.parametrize("qt,ct", KINDS)
def test_prefix(qm, dev, qt, ct, prefix_len, ws):
    """A shared prefix that ends inside a page, short and long; sequences with no tokens of their own before it."""
    run(qm, dev, [1, 40, 130, 7, 64], [1] * 5, 8, 2, 128, 16, qt, ct, prefix_len=prefix_len, ws=ws, seed=prefix_len)
    run(qm, dev, [5, 40], [5, 2], 3, 1, 64, 64, qt, ct, prefix_len=prefix_len, ws=ws, seed=prefix_len, out=F32)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_and_cut(qm, dev, D):
    """Long sequences beside short ones: cut into pieces with a workspace, whole without, and with a small one."""
    for ws in (True, False):
        run(qm, dev, [5000, 3, 700], [1, 1, 1], 4, 1, D, 64, BF16, BF16, ws=ws)
        run(qm, dev, [2100, 40], [40, 2], 4, 1, D, 64, F16, F16, ws=ws)


def test_every_workspace_size(qm, dev):
    """Any workspace serves: the pieces follow its size."""
    cache = K.Cache(60, 2, 16, 64, BF16, 0)
    start, ln, table, rest = K.batch([300, 20], [1, 1], 16, 60, 0)
    prefix = torch.tensor(rest[:17], dtype=torch.int32)
    q = queries(2, 4, 64, BF16, 1)
    kv = cache.on(qm, dev)
    want, bound = K.attention(q, cache, start, ln, table, BF16, None, prefix, 270)
    full = qm.attn_workspace(kv, 2, 2, 4, 270).numel()
    for n in (0, 256, 4096, full // 64 // 256 * 256, full // 8 // 256 * 256, full // 2 // 256 * 256, full - 256, full, full + 512):
        buf = torch.full((n + 256,), 0xFF, dtype=torch.uint8, device=dev)  # (NaN wherever it is read unwritten)
        got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), prefix=prefix.to(dev), prefix_len=270, ws=buf[:n] if n else None)
        K.check(got, want, bound, BF16)
        assert bool((buf[n:] == 0xFF).all())


@pytest.mark.parametrize("ct", [BF16, E4M3])
@pytest.mark.parametrize("order,pad", [((0, 2, 1), 0), ((1, 0, 2), 0), ((0, 1, 2), 16), ((2, 1, 0), 32)])
def test_cache_strides(qm, dev, order, pad, ct):
    run(qm, dev, [50, 3, 129], [1, 1, 1], 4, 2, 80, 32, BF16, ct, order=order, pad=pad)


def test_q_and_o_strides(qm, dev):
    """Rows of a wider matrix, at any element; nothing else is written."""
    cache = K.Cache(20, 2, 16, 64, BF16, 3)
    start, ln, table, _ = K.batch([30, 70, 17], [2, 1, 3], 16, 20, 3)
    q = queries(6, 4, 64, BF16, 4)
    kv = cache.on(qm, dev)
    args = (kv, ln.to(dev), table.to(dev))
    want = qm.attn_prefix(q.to(dev), *args, start=start.to(dev))
    for off in (8, 3):
        wide = torch.full((6, 400), 9.0, dtype=BF16, device=dev)
        rows = wide.as_strided((6, 4, 64), (400, 64, 1), off)
        rows.copy_(q)
        got = torch.full((7, 300), -3.0, dtype=BF16, device=dev)
        qm.attn_prefix(rows, *args, start=start.to(dev), o=got.as_strided((6, 4, 64), (300, 64, 1), off))
        assert torch.equal(got[:6, off:off + 256].reshape(6, 4, 64), want)
        assert bool((got[6] == -3).all()) and bool((got[:, :off] == -3).all()) and bool((got[:, off + 256:] == -3).all())


def test_rows_of_no_sequence_stay(qm, dev):
    """Rows before the first sequence and behind the last one are left as they were, whatever the workspace."""
    cache = K.Cache(12, 1, 16, 64, BF16, 5)
    _, ln, table, _ = K.batch([30, 70], [2, 3], 16, 12, 5)
    start = torch.tensor([1, 3, 6], dtype=torch.int32)
    q = queries(9, 2, 64, BF16, 6)
    want, bound = K.attention(q, cache, start, ln, table, BF16)
    kv = cache.on(qm, dev)
    for ws in (None, qm.attn_workspace(kv, 9, 2, 2)):
        o = torch.full((9, 2, 64), 5.0, dtype=BF16, device=dev)
        qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), o=o, ws=ws)
        K.check(o, want, bound, BF16)
        assert bool((o[0] == 5).all()) and bool((o[6:] == 5).all())


@pytest.mark.parametrize("ws", [True, False])
def test_empty_rows_are_zeros(qm, dev, ws):
    """More rows than the sequence has tokens, no tokens at all, lengths below zero: rows that see no key are zeros; with a prefix they see it."""
    cache = K.Cache(30, 1, 16, 64, F16, 5)
    start = torch.tensor([0, 4, 5, 6, 6], dtype=torch.int32)
    ln = torch.tensor([2, 0, -7, 0], dtype=torch.int32)
    table = torch.tensor([[3], [4], [5], [6]], dtype=torch.int32)
    q = queries(6, 2, 64, F16, 6)
    kv = cache.on(qm, dev)
    w = qm.attn_workspace(kv, 6, 4, 2, 400) if ws else None
    got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=w)
    assert not got[:2].any() and not got[4:].any() and got[2:4].all()
    K.check(got, *K.attention(q, cache, start, ln, table, F16), F16)
    prefix = torch.arange(4, 29, dtype=torch.int32)
    got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=w, prefix=prefix.to(dev), prefix_len=390)
    K.check(got, *K.attention(q, cache, start, ln, table, F16, None, prefix, 390), F16)


@pytest.mark.parametrize("ct", [BF16, F16, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_places_may_hold_anything(qm, dev, bad, ct):
    """NaN and infinities behind a sequence, behind a prefix, in spare pages and in later tokens of the same call: no effect on rows that do
    not see them; rows that see a value of infinity or NaN have it."""
    cache = K.Cache(40, 1, 16, 128, ct, 7)
    start, ln, table, rest = K.batch([37, 90], [5, 1], 16, 40, 7)
    prefix = torch.tensor(rest[:20], dtype=torch.int32)
    qt = BF16 if ct == E4M3 else ct
    q = queries(6, 3, 128, qt, 8)
    want, bound = K.attention(q, cache, start, ln, table, qt, None, prefix, 310)
    put = math.nan if ct == E4M3 else bad
    for t in cache.data:
        raw = t.view(torch.uint8) if ct == E4M3 else t
        val = 0x7F if ct == E4M3 else put
        for b, n in enumerate(ln.tolist()):
            raw[int(table[b, n // 16]), :, n % 16:] = val
        raw[rest[19], :, 310 - 19 * 16:] = val
        for p in rest[20:]:
            raw[p] = val
    for s in cache.scales:
        if s is not None:
            for b, n in enumerate(ln.tolist()):
                s[int(table[b, n // 16]), :, n % 16:] = bad
    args = lambda kv: (q.to(dev), kv, ln.to(dev), table.to(dev))  # noqa: E731
    more = dict(start=start.to(dev), prefix=prefix.to(dev), prefix_len=310)
    kv = cache.on(qm, dev)
    for ws in (None, qm.attn_workspace(kv, 6, 2, 3, 310)):
        K.check(qm.attn_prefix(*args(kv), ws=ws, **more), want, bound, qt)
    # the last two of the five new tokens: the first three rows do not see them, and the other sequence does not
    page, at = int(table[0, 35 // 16]), 35 % 16
    v = cache.data[1].view(torch.uint8) if ct == E4M3 else cache.data[1]
    v[page, 0, at, 5] = 0x7F if ct == E4M3 else bad
    k = cache.data[0].view(torch.uint8) if ct == E4M3 else cache.data[0]
    k[page, 0, at + 1, 3] = 0x7F if ct == E4M3 else bad
    kv = cache.on(qm, dev)
    for ws in (None, qm.attn_workspace(kv, 6, 2, 3, 310)):
        got = qm.attn_prefix(*args(kv), ws=ws, **more).cpu()
        keep = torch.tensor([0, 1, 2, 5])
        K.check(got[keep], want[keep], bound[keep], qt)
        assert not torch.isfinite(got[3, :, 5].float()).any()
        # (a key of plus infinity: a logit of plus infinity, whose softmax is NaN, or of minus infinity, whose weight is zero)
        sees = torch.ones(3, dtype=torch.bool) if math.isnan(put) else q[4, :, 3] > 0
        assert torch.isnan(got[4]).all(1).equal(sees) and torch.isfinite(got[4, ~sees, 6:].float()).all()
        off = (got[3].double() - want[3]).abs()[:, 6:]
        assert bool(torch.isfinite(off).all())  # (only the value's own element)


def test_bad_pages_and_lengths(qm, dev):
    """Page numbers outside the cache mask their keys; lengths beyond the table end with it; nothing outside is read."""
    cache = K.Cache(10, 2, 16, 64, BF16, 9)
    table = torch.tensor([[1, -1, 3, 2 ** 31 - 1], [10, 4, -2 ** 31, 5], [-1, -5, 99, 10]], dtype=torch.int32)
    ln = torch.tensor([60, 2 ** 31 - 1, 64], dtype=torch.int32)
    start = torch.tensor([0, 2, 4, 5], dtype=torch.int32)
    prefix = torch.tensor([7, -1] + [8] * 15 + [10], dtype=torch.int32)
    q = queries(5, 2, 64, BF16, 10)
    kv = cache.on(qm, dev)
    for ws in (None, qm.attn_workspace(kv, 5, 3, 2, 288)):
        got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=ws)
        K.check(got, *K.attention(q, cache, start, ln, table, BF16), BF16)
        assert not got[4].any()
        got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=ws, prefix=prefix.to(dev), prefix_len=288)
        K.check(got, *K.attention(q, cache, start, ln, table, BF16, None, prefix, 288), BF16)


def test_starts_that_are_no_list(qm, dev):
    """Rows outside 0..T and descending lists: no sequence has rows that the call has not, and nothing else is written."""
    cache = K.Cache(10, 1, 16, 64, BF16, 9)
    kv = cache.on(qm, dev)
    ln = torch.full((3,), 20, dtype=torch.int32, device=dev)
    table = torch.tensor([[1, 2], [3, 4], [5, 6]], dtype=torch.int32, device=dev)
    q = queries(4, 1, 64, BF16, 10).to(dev)
    for start in ([-5, 2, 9, 40], [3, 2, 1, 0], [4, 4, 4, 4], [0, 4, 0, 4]):
        for ws in (None, qm.attn_workspace(kv, 4, 3, 1)):
            buf = torch.full((6, 1, 64), 3.0, dtype=BF16, device=dev)
            qm.attn_prefix(q, kv, ln, table, start=torch.tensor(start, dtype=torch.int32, device=dev), o=buf[1:5], ws=ws)
            assert bool((buf[0] == 3).all()) and bool((buf[5] == 3).all())


def test_scales_and_extremes(qm, dev):
    """Scales of zero and below, and logits so far apart that all but one weight vanish."""
    for scale in (0.0, -0.3, 30.0):
        run(qm, dev, [40, 100], [1, 1], 2, 1, 64, 16, F16, F16, scale=scale, out=F32)
        run(qm, dev, [40, 100], [9, 1], 2, 1, 64, 16, BF16, BF16, scale=scale)


def test_pieces_and_whole_agree_when_lengths_grow(qm, dev):
    """A captured call with sequences that grow: lengths are read at the replay; two graphs with a workspace each."""
    cache = K.Cache(80, 2, 16, 128, BF16, 11)
    start, ln, table, rest = K.batch([600, 40, 300], [1, 1, 1], 16, 70, 11, spare=4)
    prefix = torch.tensor(rest[:1] * 17, dtype=torch.int32).to(dev)
    table[:, -4:] = torch.tensor([70, 71, 72, 73], dtype=torch.int32)  # (room to grow; shared, as this only reads)
    for b, n in enumerate(ln.tolist()):
        table[b, (n + 15) // 16:] = 74
    q = queries(3, 8, 128, BF16, 12)
    kv, qd, ld, td = cache.on(qm, dev), q.to(dev), ln.to(dev), table.to(dev)
    outs, graphs = [], []
    for i in range(2):
        ws, o = qm.attn_workspace(kv, 3, 3, 8, 270), torch.empty((3, 8, 128), dtype=BF16, device=dev)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qm.attn_prefix(qd, kv, ld, td, prefix=prefix if i else None, prefix_len=270 if i else 0, o=o, ws=ws)
        outs.append((o, ws))
        graphs.append(g)
    for step in range(4):
        ld.add_(3)
        for g in graphs:
            g.replay()
        eager = [qm.attn_prefix(qd, kv, ld, td, prefix=prefix if i else None, prefix_len=270 if i else 0,
                                ws=qm.attn_workspace(kv, 3, 3, 8, 270)) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], eager[i])
            want, bound = K.attention(q, cache, start, ld.cpu(), table, BF16, None, prefix.cpu() if i else (), 270 if i else 0)
            K.check(outs[i][0], want, bound, BF16)


def test_streams(qm, dev):
    """Calls on two streams at once, a workspace each, and repeated: the same bits."""
    cache = K.Cache(80, 2, 16, 128, F16, 13)
    start, ln, table, _ = K.batch([700, 90], [3, 1], 16, 80, 13)
    q = queries(4, 4, 128, F16, 14).to(dev)
    kv = cache.on(qm, dev)
    args = (q, kv, ln.to(dev), table.to(dev))
    want = qm.attn_prefix(*args, start=start.to(dev), ws=qm.attn_workspace(kv, 4, 2, 4))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [qm.attn_prefix(*args, start=start.to(dev), ws=qm.attn_workspace(kv, 4, 2, 4)) for _ in range(3)]
    for s in streams:
        s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_caches_past_32_bit_offsets(qm, dev):
    """Pages more than 2^32 bytes into the cache."""
    D, page, HK = 128, 64, 1
    pages = (2 ** 32 + 2 ** 28) // (page * D * 2)
    k = torch.empty((pages, HK, page, D), dtype=BF16, device=dev)
    far = [pages - 1, pages // 2 + 5, 3, pages - 70]
    small = K.Cache(4, HK, page, D, BF16, 15)
    k[far] = small.data[0].to(dev)
    v = torch.empty_like(k)
    v[far] = small.data[1].to(dev)
    kv = qm.KvCache(k, v)
    q = queries(1, 2, D, BF16, 16)
    ln = torch.tensor([250], dtype=torch.int32)
    got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), torch.tensor([far], dtype=torch.int32, device=dev))
    K.check(got, *K.attention(q, small, torch.tensor([0, 1]), ln, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32), BF16), BF16)


# ---- many rows: prompts, and a prefix for the rows of a large batch
@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D,page", [(16, 16), (64, 64), (80, 16), (128, 32), (144, 16), (192, 128), (256, 16)])
def test_many_rows(qm, dev, D, page, qt, ct, out):
    """Prompts from their first token and behind others, one token among them; tiles that end inside a token's heads; whole and in pieces."""
    for ws in (True, False):
        run(qm, dev, [90, 64, 1, 333], [90, 40, 1, 70], 6, 2, D, page, qt, ct, out=out, ws=ws, seed=D)


@pytest.mark.parametrize("prefix_len", [1, 33, 100, 300])
@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_rows_behind_a_prefix(qm, dev, D, qt, ct, prefix_len):
    run(qm, dev, [70, 5], [70, 1], 5, 1, D, 16, qt, ct, prefix_len=prefix_len, seed=prefix_len)
    run(qm, dev, [66], [65], 2, 2, D, 32, qt, ct, prefix_len=prefix_len, seed=prefix_len, ws=False)


@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_prefix_of_a_large_batch(qm, dev, D, qt, ct):
    """64 rows of a key head and more: the prefix by their tiles, the sequences' own keys by themselves."""
    lens = [1 + 7 * i % 90 for i in range(30)]
    for out, n in ((None, 256), (F32, 700), (None, 1111)):
        run(qm, dev, lens, [1] * 30, 10, 2, D, 16, qt, ct, out=out, prefix_len=n, seed=n)
    run(qm, dev, lens[:23], [min(n, 3) for n in lens[:23]], 2, 2, D, 32, qt, ct, prefix_len=300, seed=1)


@pytest.mark.parametrize("rows", [63, 64, 65, 127, 128, 129, 257])
def test_around_tiles(qm, dev, rows):
    for D in (64, 128, 192):
        run(qm, dev, [rows + 3], [rows], 1, 1, D, 16, BF16, BF16, seed=rows)
        run(qm, dev, [5000], [rows], 1, 1, D, 64, F16, F16, seed=rows)


@pytest.mark.parametrize("ct", [BF16, E4M3])
@pytest.mark.parametrize("order,pad", [((0, 2, 1), 0), ((1, 0, 2), 16)])
def test_many_rows_strides(qm, dev, order, pad, ct):
    run(qm, dev, [150, 3, 129], [90, 3, 100], 4, 2, 80, 32, BF16, ct, order=order, pad=pad)


@pytest.mark.parametrize("ct", [BF16, F16, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_many_rows_masked_places(qm, dev, bad, D, ct):
    """NaN and infinities where no row sees them, and values of them that some of a tile's rows see and others do not."""
    cache = K.Cache(40, 1, 16, D, ct, 7)
    start, ln, table, rest = K.batch([137, 90], [70, 60], 16, 40, 7)
    prefix = torch.tensor(rest[:5], dtype=torch.int32)
    qt = BF16 if ct == E4M3 else ct
    q = queries(130, 2, D, qt, 8)
    want, bound = K.attention(q, cache, start, ln, table, qt, None, prefix, 77)
    put = lambda t, at, val: t.view(torch.uint8).__setitem__(at, 0x7F) if ct == E4M3 else t.__setitem__(at, val)  # noqa: E731
    for t in cache.data:
        for b, n in enumerate(ln.tolist()):
            put(t, (int(table[b, n // 16]), slice(None), slice(n % 16, 16)), bad)
        put(t, (rest[4], slice(None), slice(77 - 64, 16)), bad)
        for p in rest[5:]:
            put(t, p, bad)
    kv = cache.on(qm, dev)
    more = dict(start=start.to(dev), prefix=prefix.to(dev), prefix_len=77)
    both = (None, qm.attn_workspace(kv, 130, 2, 2, 77))
    for ws in both:
        K.check(qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), ws=ws, **more), want, bound, qt)
    # values of the first sequence's tokens 100 and 118: its rows are tokens 67 to 136
    for token, d in ((100, 5), (118, D - 1)):
        put(cache.data[1], (int(table[0, token // 16]), 0, token % 16, d), bad)
    kv = cache.on(qm, dev)
    for ws in both:
        got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), ws=ws, **more).cpu()
        hit = torch.zeros((130, 2, D), dtype=torch.bool)
        hit[100 - 67:70, :, 5] = True
        hit[118 - 67:70, :, D - 1] = True
        assert not torch.isfinite(got[hit].float()).any()
        assert ct == E4M3 or torch.equal(got[hit], torch.full_like(got[hit], bad)) or math.isnan(bad)
        K.check(torch.where(hit, want.to(qt), got), want, bound, qt)


@pytest.mark.parametrize("rows", [5, 80])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_scales_of_masked_places(qm, dev, bad, D, rows):
    """An 8-bit cache's scales of NaN and infinities where no row sees them, and of a key and a value that the last rows see and the others do not."""
    cache = K.Cache(20, 1, 16, D, E4M3, 7)
    start, ln, table, rest = K.batch([150], [rows], 16, 20, 7)
    prefix = torch.tensor(rest[:3], dtype=torch.int32)
    q = queries(rows, 2, D, BF16, 8)
    want, bound = K.attention(q, cache, start, ln, table, BF16, None, prefix, 37)
    for s in cache.scales:
        s[int(table[0, 150 // 16]), :, 150 % 16:] = bad
        s[rest[2], :, 37 - 32:] = bad
        s[rest[3:]] = bad
    more = dict(start=start.to(dev), prefix=prefix.to(dev), prefix_len=37)
    for which, token in ((None, 150), (1, 148), (0, 147)):
        if which is not None:
            cache.scales[which][int(table[0, token // 16]), 0, token % 16] = bad
        kv = cache.on(qm, dev)
        for ws in (None, qm.attn_workspace(kv, rows, 1, 2, 37)):
            got = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), ws=ws, **more).cpu()
            n = rows - (150 - token)  # rows that do not see it
            K.check(got[:n], want[:n], bound[:n], BF16)
            if which == 1:
                assert not torch.isfinite(got[n:].float()).any(2).any()


@pytest.mark.parametrize("HK,G,new,lens,prefix_len", [(2, 4, [300, 70], [900, 2000], 0), (64, 1, [1100], [1100], 0), (2, 16, [1] * 100, [40 + i for i in range(100)], 20100)])
def test_many_rows_on_two_streams(qm, dev, HK, G, new, lens, prefix_len):
    """Pieces, tiles of a last round that are cut, and a prefix in a launch of its own: calls on two streams at once, a workspace each, and repeated: the
    same bits."""
    cache = K.Cache(sum((n + 63) // 64 for n in lens) + (prefix_len + 63) // 64, HK, 64, 128, BF16, 13)
    start, ln, table, rest = K.batch(lens, new, 64, cache.pages, 13)
    T = int(start[-1])
    q = queries(T, HK * G, 128, BF16, 14).to(dev)
    kv = cache.on(qm, dev)
    prefix = torch.tensor(rest[:(prefix_len + 63) // 64], dtype=torch.int32).to(dev)
    args, more = (q, kv, ln.to(dev), table.to(dev)), dict(start=start.to(dev), prefix=prefix if prefix_len else None, prefix_len=prefix_len)
    space = lambda: qm.attn_workspace(kv, T, len(lens), HK * G, prefix_len)  # noqa: E731
    want = qm.attn_prefix(*args, **more, ws=space())
    torch.cuda.synchronize()
    streams, got, kept = [torch.cuda.Stream() for _ in range(2)], [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            kept.append(space())
            got += [qm.attn_prefix(*args, **more, ws=kept[-1]) for _ in range(4)]
    for s in streams:
        s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_many_rows_bad_pages(qm, dev):
    cache = K.Cache(10, 2, 16, 128, BF16, 9)
    table = torch.tensor([[1, -1, 3, 2 ** 31 - 1, 4, 5], [10, 4, -2 ** 31, 5, 6, 7]], dtype=torch.int32)
    ln = torch.tensor([90, 2 ** 31 - 1], dtype=torch.int32)
    start = torch.tensor([0, 100, 150], dtype=torch.int32)  # (ten rows of the first sequence see none of its keys)
    prefix = torch.tensor([7, -1, 8, 10], dtype=torch.int32)
    q = queries(152, 2, 128, BF16, 10)
    kv = cache.on(qm, dev)
    for ws in (None, qm.attn_workspace(kv, 152, 2, 2, 60)):
        for n in (0, 60):
            o = torch.full((152, 2, 128), 4.0, dtype=BF16, device=dev)
            qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=ws, prefix=prefix.to(dev) if n else None, prefix_len=n, o=o)
            want, bound = K.attention(q, cache, start, ln, table, BF16, None, prefix if n else (), n)
            K.check(o[:150], want[:150], bound[:150], BF16)
            assert bool((o[150:] == 4).all()) and (n or not o[:10].any())


def test_many_rows_replayed(qm, dev):
    """A captured prompt and a captured decode step of a large batch behind a prefix, replayed with other lengths."""
    cache = K.Cache(90, 1, 16, 64, BF16, 11)
    kv = cache.on(qm, dev)
    pages = torch.randperm(89, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    table = pages[20:80].reshape(30, 2).contiguous()
    start = torch.tensor([0, 70], dtype=torch.int32)
    calls = []
    for lens, st, n, tab, rows in ((torch.tensor([90]), start, 0, pages[:8].reshape(1, 8).contiguous(), 70), (torch.arange(30) % 20 + 1, None, 290, table, 30)):
        q = queries(rows, 4, 64, BF16, n)
        ld = lens.to(torch.int32).to(dev)
        ws, o = qm.attn_workspace(kv, rows, len(lens), 4, n), torch.empty((rows, 4, 64), dtype=BF16, device=dev)
        kw = dict(start=None if st is None else st.to(dev), prefix=pages[:19].to(dev) if n else None, prefix_len=n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        qd, td = q.to(dev), tab.to(dev)
        with torch.cuda.graph(g):
            qm.attn_prefix(qd, kv, ld, td, o=o, ws=ws, **kw)
        calls.append((q, ld, tab, st, n, o, g, qd, td, kw, ws))
    for step in range(3):
        for q, ld, tab, st, n, o, g, qd, td, kw, ws in calls:
            ld.add_(4)
            g.replay()
            eager = qm.attn_prefix(qd, kv, ld, td, ws=qm.attn_workspace(kv, q.shape[0], len(ld), 4, n), **kw)
            torch.cuda.synchronize()
            assert torch.equal(o, eager)
            st = torch.arange(q.shape[0] + 1) if st is None else st
            K.check(o, *K.attention(q, cache, st, ld.cpu(), tab, BF16, None, pages[:19] if n else (), n), BF16)


@pytest.mark.parametrize("D,HK,G,rows,lens", [(64, 64, 1, [1100], [1100]), (16, 70, 2, [300, 200, 60], [300, 1500, 70]), (256, 33, 2, [520], [700]),
                                              (128, 64, 1, [128, 1], [900, 5])])
def test_last_round_of_tiles(qm, dev, D, HK, G, rows, lens):
    """More row tiles than the GPU takes at once: those behind the last whole round are cut. Rows of many sequences, a few of whose results are
    looked at; rows behind the last one stay; the workspace may hold anything, and any size of it serves."""
    page, T = 32, max(sum(rows), 1100)
    cache = K.Cache(sum((n + page - 1) // page for n in lens) + 2, HK, page, D, BF16, 21)
    start, ln, table, rest = K.batch(lens, rows, page, cache.pages, 21)
    q = queries(T, HK * G, D, BF16, 22)
    kv = cache.on(qm, dev)
    some, see, of = [], [], []
    for b, n in enumerate(rows):
        for t in {0, 1, n // 3, n // 2, n - 2, n - 1} & set(range(n)):
            some.append(int(start[b]) + t)
            see.append(lens[b] - n + t + 1)
            of.append(b)
    want, bound = K.attention(q[some], cache, torch.arange(len(some) + 1), torch.tensor(see), table[of], BF16)
    full = qm.attn_workspace(kv, T, len(rows), HK * G).numel()
    outs = []
    for n in (full, 0, full // 2 // 256 * 256, full + 256):
        ws = torch.full((max(n, 256),), 0xFF, dtype=torch.uint8, device=dev)
        o = torch.full((T, HK * G, D), 3.0, dtype=BF16, device=dev)
        qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), o=o, ws=ws[:n] if n else None)
        K.check(o[some], want, bound, BF16)
        assert bool((o[sum(rows):] == 3).all())
        outs.append(o)
    # (cut or whole, every row is within two roundings of the other)
    a, b = (outs[i][:sum(rows)].double() for i in (0, 1))
    assert bool(((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -8).all())


def shared(qm, dev, qt, ct, D, B, HQ, HK, n, prefix_len, page, out=None, sizes=(1.0,)):
    """A batch of n tokens a sequence behind a prefix: a few rows of the result against the plain form, all against the call without a workspace."""
    lens = [n + 9 * i % 70 for i in range(B)]
    cache = K.Cache(sum((m + page - 1) // page for m in lens) + (prefix_len + page - 1) // page, HK, page, D, ct, 31)
    start, ln, table, rest = K.batch(lens, [n] * B, page, cache.pages, 31)
    prefix = torch.tensor(rest, dtype=torch.int32)
    q, out = queries(n * B, HQ, D, qt, 32), out or qt
    kv = cache.on(qm, dev)
    of = [0, B // 2, B - 1]
    some, see = [n * b + (n - 1) * (b % 2) for b in of], [lens[b] - n + 1 + (n - 1) * (b % 2) for b in of]
    want, bound = K.attention(q[some], cache, torch.arange(4), torch.tensor(see), table[of], out, None, prefix, prefix_len)
    full = qm.attn_workspace(kv, n * B, B, HQ, prefix_len).numel()
    args = (q.to(dev), kv, ln.to(dev), table.to(dev))
    more = dict(start=None if n == 1 else start.to(dev), prefix=prefix.to(dev), prefix_len=prefix_len, out=out)
    alone = qm.attn_prefix(*args, **more)
    K.check(alone[some], want, bound, out)
    for part in sizes:
        ws = torch.full((int(full * part) // 256 * 256,), 0xFF, dtype=torch.uint8, device=dev)  # (NaN wherever it is read unwritten)
        got = qm.attn_prefix(*args, **more, ws=ws)
        K.check(got[some], want, bound, out)
        a, b = got.double(), alone.double()
        assert bool(((a - b).abs() <= (2.0 ** -6 if out != F32 else 2.0 ** -12) * (a.abs() + 1)).all())
    return full


@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D,B,HQ,n", [(64, 20, 6, 1), (80, 9, 4, 2), (128, 11, 8, 1), (256, 6, 24, 2)])
def test_shared_prefix(qm, dev, D, B, HQ, n, qt, ct):
    """A prefix that is worth being read once (32 MB less), in the sequences' own launch."""
    unit = (B - 1) * 2 * D * (2 if ct == E4M3 else 4)
    prefix_len = int(3.2e7 / unit) + 45
    for out in (None, F32):
        full = shared(qm, dev, qt, ct, D, B, HQ, 2, n, prefix_len, 32, out, (1.0, 0.5, 0.1))
    assert full != qm.attn_workspace(K.Cache(1, 2, 32, D, ct, 0).on(qm, dev), n * B, B, HQ, prefix_len - 46).numel()  # (below the bytes: another plan)


@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D,T", [(64, 256), (96, 192), (128, 128), (256, 64)])
def test_shared_prefix_by_large_tiles(qm, dev, D, T, qt, ct):
    """One of so many products that it has a launch of its own."""
    prefix_len = int((6e9 if ct == E4M3 else 4e9) / (T * 32 * D)) + 77
    shared(qm, dev, qt, ct, D, T, 32, 2, 1, prefix_len, 64, sizes=(1.0, 0.3))
    shared(qm, dev, qt, ct, D, T // 3, 32, 2, 3, prefix_len, 64, F32)


def test_many_rows_scales(qm, dev):
    for scale in (0.0, -0.3, 30.0):
        for D in (64, 128, 256):
            run(qm, dev, [130, 70], [60, 40], 2, 1, D, 16, F16, F16, scale=scale, out=F32)
            run(qm, dev, [130, 70], [60, 40], 2, 1, D, 16, BF16, E4M3, scale=scale)


def test_many_rows_q_and_o_strides(qm, dev):
    """Rows of a wider matrix, at any element; nothing else is written."""
    cache = K.Cache(20, 2, 16, 128, BF16, 3)
    start, ln, table, _ = K.batch([90, 70], [66, 41], 16, 20, 3)
    q = queries(107, 4, 128, BF16, 4)
    kv = cache.on(qm, dev)
    args = (kv, ln.to(dev), table.to(dev))
    for out in (BF16, F32):
        want = qm.attn_prefix(q.to(dev), *args, start=start.to(dev), out=out)
        for off in (8, 3):
            wide = torch.full((107, 700), 9.0, dtype=BF16, device=dev)
            rows = wide.as_strided((107, 4, 128), (700, 128, 1), off)
            rows.copy_(q)
            got = torch.full((108, 601), -3.0, dtype=out, device=dev)
            for ws in (None, qm.attn_workspace(kv, 107, 2, 4)):
                o = qm.attn_prefix(rows, *args, start=start.to(dev), o=got.as_strided((107, 4, 128), (601, 128, 1), off), ws=ws)
                if ws is None:
                    assert torch.equal(o, want)
            assert bool((got[107] == -3).all()) and bool((got[:, :off] == -3).all()) and bool((got[:, off + 512:] == -3).all())


@pytest.mark.parametrize("rows", [1, 70])
def test_lengths_of_any_value(qm, dev, rows):
    """The least and the largest lengths: none of the keys, and all that the table holds."""
    cache = K.Cache(10, 1, 16, 64, BF16, 5, mean=True)
    kv = cache.on(qm, dev)
    table = torch.tensor([[1, 2, 3], [4, 5, 6], [7, 8, 9]], dtype=torch.int32)
    ln = torch.tensor([-2 ** 31, 2 ** 31 - 1, -2 ** 31 + 5], dtype=torch.int32)
    start = torch.tensor([0, 1, 2, 3], dtype=torch.int32) * rows
    q = queries(3 * rows, 2, 64, BF16, 6)
    args = (q.to(dev), kv, ln.to(dev), table.to(dev))
    want, bound = K.attention(q, cache, start, ln.clamp(min=0), table, BF16)
    for ws in (None, qm.attn_workspace(kv, 3 * rows, 3, 2)):
        o = qm.attn_prefix(*args, start=start.to(dev), ws=ws)
        K.check(o, want, bound, BF16)
        assert not o[:rows].any() and not o[2 * rows:].any() and o[rows:2 * rows].any(2).all()
    sel = qm.select_pages(*args, 2, start=start.to(dev))
    assert bool((sel[:rows] == -1).all()) and bool((sel[2 * rows:] == -1).all()) and bool((sel[rows:2 * rows] >= 0).all())
    o = qm.attn_pages(*args, torch.tensor([0, 1, 2], dtype=torch.int32, device=dev).expand(3 * rows, 1, 3).contiguous(), start=start.to(dev))
    K.check(o, want, bound, BF16)


@pytest.mark.parametrize("B,HK,G,most,prefix_len", [(300, 4, 2, 1, 0), (1100, 1, 20, 1, 0), (400, 4, 3, 3, 0), (150, 8, 40, 2, 0), (300, 4, 4, 2, 700),
                                                   (1100, 1, 2, 2, 300)])
def test_batches_of_many_sequences(qm, dev, B, HK, G, most, prefix_len):
    """More sequences than a wave adds up at once, some without rows; a few rows of the result are looked at, rows of no sequence stay."""
    g = torch.Generator().manual_seed(B)
    new = [1] * B if most == 1 else torch.randint(0, most + 1, (B,), generator=g).tolist()
    lens = [max(n, 1) + i % 37 for i, n in enumerate(new)]
    cache = K.Cache(4 * B + 60, HK, 16, 64, BF16, 1)
    start, ln, table, rest = K.batch(lens, new, 16, cache.pages, 2)
    prefix = torch.tensor(rest[:(prefix_len + 15) // 16], dtype=torch.int32)
    T = int(start[-1])
    q = queries(T + 3, HK * G, 64, BF16, 3)
    kv = cache.on(qm, dev)
    some = sorted({0, 1, T // 3, T // 2, T - 2, T - 1})
    of = [int(torch.searchsorted(start[1:], t, right=True)) for t in some]
    see = [lens[b] - (int(start[b + 1]) - t) + 1 for t, b in zip(some, of)]
    want, bound = K.attention(q[some], cache, torch.arange(len(some) + 1), torch.tensor(see), table[of], BF16, None, prefix, prefix_len)
    outs = []
    for ws in (None, qm.attn_workspace(kv, T + 3, B, HK * G, prefix_len)):
        if most == 1:
            o = qm.attn_prefix(q[:T].to(dev), kv, ln.to(dev), table.to(dev), ws=ws)
        else:
            o = torch.full((T + 3, HK * G, 64), 5.0, dtype=BF16, device=dev)
            qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), ws=ws, o=o, prefix=prefix.to(dev), prefix_len=prefix_len)
            assert bool((o[T:] == 5).all())
        K.check(o[some], want, bound, BF16)
        outs.append(o[:T].double())
    a, b = outs
    assert bool(((a - b).abs() <= 2.0 ** -6 * (a.abs() + 1)).all()) and bool(a.any(2).all())


# ---- chosen pages
@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("qt,ct", KINDS)
@pytest.mark.parametrize("D,page,G", [(64, 16, 4), (128, 32, 1), (80, 64, 17), (256, 16, 6)])
def test_chosen_pages(qm, dev, D, page, G, qt, ct, ws):
    """Any list of pages: none, beyond the row's own place, in any order, twice, outside the table."""
    HK = 2
    cache = K.Cache(40, HK, page, D, ct, D)
    start, ln, table, _ = K.batch([5 * page + 3, page, 9 * page], [3, 1, 2], page, 40, D)
    g = torch.Generator().manual_seed(D)
    sel = torch.randint(-1, table.shape[1] + 1, (6, HK, 7), generator=g, dtype=torch.int32)
    sel[0, 0] = -1
    sel[1, 1] = torch.tensor([0, 0, 5, 5, -9, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    q = queries(6, G * HK, D, qt, 3)
    for out in (qt, F32):
        kv = cache.on(qm, dev)
        got = qm.attn_pages(q.to(dev), kv, ln.to(dev), table.to(dev), sel.to(dev), start=start.to(dev), out=out,
                            ws=qm.attn_workspace(kv, 6, 6, G * HK) if ws else None)
        K.check(got, *K.attention(q, cache, start, ln, table, out, sel=sel), out)
        assert not got[0, :G].any()


def test_all_pages_chosen_is_everything(qm, dev):
    cache = K.Cache(70, 2, 32, 128, BF16, 1)
    start, ln, table, _ = K.batch([1000, 700, 33], [1, 1, 1], 32, 70, 1, spare=0)
    q = queries(3, 8, 128, BF16, 2).to(dev)
    kv = cache.on(qm, dev)
    n = table.shape[1]
    sel = torch.arange(n, dtype=torch.int32).expand(3, 2, n).contiguous().to(dev)
    want, bound = K.attention(q.cpu(), cache, start, ln, table, BF16)
    for ws in (None, qm.attn_workspace(kv, 3, 3, 8)):
        K.check(qm.attn_pages(q, kv, ln.to(dev), table.to(dev), sel, ws=ws), want, bound, BF16)
