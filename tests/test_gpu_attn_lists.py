"""Attention over a paged cache with lists of rows that are no batch, and a workspace that holds anything: some rows' pieces are nobody's, and the join takes no
word of such a slot unseen. (Which rows those are is worked out in tests/test_attn_split.py.)"""
import pytest
import torch

from tests import kv_plain as K

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("words", ["ones", "least", "largest", "random"])
@pytest.mark.parametrize("prefix_len", [0, 1000])
def test_descending_lists(qm, dev, words, prefix_len):
    """Nothing outside o is written, and o is what the call's rows may be: the call ends."""
    T, HQ, HK, D = 90, 8, 2, 128
    cache = K.Cache(40, HK, 16, D, BF16, 1)
    kv = cache.on(qm, dev)
    q = torch.randn((T, HQ, D), generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    prefix = (torch.arange(63, dtype=torch.int32) % 40).to(dev)
    for start in ([0, 90] * 8, [90, 0, 90, 0, 0], [-5, 90, 20, 2 ** 31 - 1, -2 ** 31, 7], [89, 0, 90] * 30):
        B = len(start) - 1
        ln = torch.full((B,), 3000, dtype=torch.int32, device=dev)
        table = (torch.arange(B * 190, dtype=torch.int32).view(B, 190) % 40).to(dev)
        n = qm.attn_workspace(kv, T, B, HQ, prefix_len).numel()
        g = torch.Generator().manual_seed(3)
        fill = {"ones": torch.full((n // 4,), -1), "least": torch.full((n // 4,), -2 ** 31), "largest": torch.full((n // 4,), 2 ** 31 - 1),
                "random": torch.randint(-2 ** 31, 2 ** 31, (n // 4,), generator=g)}[words]
        buf = torch.zeros((n + 512,), dtype=torch.uint8, device=dev)
        buf[:n] = fill.to(torch.int32).to(dev).view(torch.uint8)
        buf[n:] = 77
        o = torch.full((T + 2, HQ, D), 3.0, dtype=BF16, device=dev)
        qm.attn_prefix(q, kv, ln, table, start=torch.tensor(start, dtype=torch.int32, device=dev), prefix=prefix if prefix_len else None, prefix_len=prefix_len,
                       o=o[1:T + 1], ws=buf[:n])
        torch.cuda.synchronize()
        assert bool((o[0] == 3).all()) and bool((o[T + 1] == 3).all()) and bool((buf[n:] == 77).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("prefix_len,rows", [(0, 1), (0, 3), (2000, 1)])
def test_values_of_vanishing_weight(qm, dev, bad, prefix_len, rows):
    """A value that is not finite, of a key that rows see with a weight of e^-400: 0 times it in 32 bits, in the limit it itself, never a finite result. In
    pieces as whole."""
    D, B = 128, 40 if prefix_len else 1
    own = 3000 if not prefix_len else 20
    cache = K.Cache((own + 15) // 16 * B + (prefix_len + 15) // 16, 1, 16, D, BF16, 1)
    start, ln, table, rest = K.batch([own] * B, [rows] * B, 16, cache.pages, 1, spare=0)
    q = torch.zeros((rows * B, 2, D))
    q[..., 0] = 8.0
    cache.data[0][..., 0] = 0.0
    pages = rest if prefix_len else table[0].tolist()
    for p in pages[:20]:  # (the first keys: far below the others)
        cache.data[0][p, :, :, 0] = -50.0
    cache.data[1][pages[3], 0, 5, 7] = bad
    kv, qd = cache.on(qm, dev), q.to(BF16).to(dev)
    prefix = torch.tensor(rest, dtype=torch.int32).to(dev) if prefix_len else None
    more = dict(start=start.to(dev), prefix=prefix, prefix_len=prefix_len, scale=1.0)
    for ws in (None, qm.attn_workspace(kv, rows * B, B, 2, prefix_len)):
        o = qm.attn_prefix(qd, kv, ln.to(dev), table.to(dev), ws=ws, **more).float()
        odd = ~torch.isfinite(o)
        assert bool(odd[..., 7].all()) and not odd[..., :7].any() and not odd[..., 8:].any()


@pytest.mark.parametrize("qt,ct", [(BF16, BF16), (torch.float16, torch.float16), (BF16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("D", [64, 256])
def test_scale_of_zero(qm, dev, D, qt, ct):
    """Weights are equal whatever q holds; a q that is not finite makes its row NaN, as 0 times it. Rows of any number, and a prefix that a large batch shares."""
    for rows, B, prefix_len in ((3, 1, 0), (100, 2, 50), (1, 140, 2100 if D == 256 else 8000)):
        cache = K.Cache((120 + 15) // 16 * B + (prefix_len + 15) // 16, 2, 16, D, ct, 1)
        start, ln, table, rest = K.batch([120] * B, [rows] * B, 16, cache.pages, 1)
        q = torch.randn((rows * B, 8, D), generator=torch.Generator().manual_seed(2)).to(qt)
        odd = torch.zeros((rows * B, 8), dtype=torch.bool)
        for t, h, d, v in ((0, 1, 5, float("inf")), (rows * B - 1, 7, D - 1, float("-inf")), (rows * B // 2, 4, 0, float("nan"))):
            q[t, h, d] = v
            odd[t, h] = True
        some = sorted({0, rows * B // 2, rows * B - 1, rows * B // 3})
        of = [t // rows for t in some]
        prefix = torch.tensor(rest[:(prefix_len + 15) // 16], dtype=torch.int32)
        clean = torch.where(odd[..., None], torch.zeros_like(q), q)
        want, bound = K.attention(clean[some], cache, torch.arange(len(some) + 1), torch.tensor([120 - rows + 1 + t % rows for t in some]), table[of], qt, 0.0, prefix, prefix_len)
        kv = cache.on(qm, dev)
        for ws in (None, qm.attn_workspace(kv, rows * B, B, 8, prefix_len)):
            o = qm.attn_prefix(q.to(dev), kv, ln.to(dev), table.to(dev), start=start.to(dev), prefix=prefix.to(dev) if prefix_len else None, prefix_len=prefix_len, scale=0.0, ws=ws)
            assert torch.equal(torch.isnan(o).all(2).cpu(), odd) and torch.equal(torch.isnan(o).any(2).cpu(), odd)
            K.check(torch.where(odd[some][..., None].to(dev), want.to(qt).to(dev), o[some]), want, bound, qt)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_of_vanishing_weight_in_a_last_round(qm, dev, bad):
    """The same by large tiles that are cut behind the last whole round of work-groups: rows that see the key have no finite result, the others have theirs."""
    D, HK, T, at = 128, 64, 1100, 53
    cache = K.Cache((T + 15) // 16, HK, 16, D, BF16, 1)
    start, ln, table, _ = K.batch([T], [T], 16, cache.pages, 1, spare=0)
    q = torch.zeros((T, HK, D))
    q[..., 0] = 8.0
    cache.data[0][..., 0] = 0.0
    for p in table[0, :20].tolist():
        cache.data[0][p, :, :, 0] = -50.0
    cache.data[1][int(table[0, at // 16]), :, at % 16, 7] = bad
    kv, qd = cache.on(qm, dev), q.to(BF16).to(dev)
    for ws in (None, qm.attn_workspace(kv, T, 1, HK)):
        odd = ~torch.isfinite(qm.attn_prefix(qd, kv, ln.to(dev), table.to(dev), start=start.to(dev), scale=1.0, ws=ws).float())
        assert bool(odd[at:, :, 7].all()) and not odd[:at].any() and not odd[..., :7].any() and not odd[..., 8:].any()
