"""The choice of pages on the GPU against its 64-bit form (tests/kv_plain.py), and a run of the cache's operators together."""
import math

import pytest
import torch

from tests import fp8_plain as P
from tests import kv_plain as K
from tests.test_gpu_kv_append import inv_freq

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def queries(T, HQ, D, dtype, seed):
    return torch.randn((T, HQ, D), generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("qt", [BF16, F16])
@pytest.mark.parametrize("D,page,HK,G,k,first,last", [
    (64, 16, 2, 4, 5, 1, 1), (128, 32, 1, 1, 1, 0, 1), (80, 64, 3, 9, 8, 0, 3), (256, 16, 1, 6, 20, 2, 2), (16, 16, 2, 17, 4, 1, 3), (128, 16, 2, 8, 64, 1, 2)])
def test_pages(qm, dev, D, page, HK, G, k, first, last, qt):
    lens, new = [37 * page + 3, page, 1, 5 * page, 80 * page - 1], [3, 1, 1, 40, 2]
    cache = K.Cache(140, HK, page, D, BF16, D + k, mean=True)
    start, ln, table, _ = K.batch(lens, new, page, 140, D)
    T = int(start[-1])
    q = queries(T, G * HK, D, qt, k)
    kv = cache.on(qm, dev)
    got = qm.select_pages(q.to(dev), kv, ln.to(dev), table.to(dev), k, start=start.to(dev), first=first, last=last)
    assert torch.equal(got.cpu(), K.chosen(q, cache, start, ln, table, k, first, last))


@pytest.mark.parametrize("n", [255, 256, 257, 700, 5000])
def test_long_tables(qm, dev, n):
    """Pages beyond one work-group's, k of one to nearly all."""
    cache = K.Cache(n, 1, 16, 32, F16, n, mean=True)
    start, ln, table, _ = K.batch([16 * n - 5], [1], 16, n, n)
    q = queries(1, 2, 32, F16, 1)
    kv = cache.on(qm, dev)
    for k in (1, 2, 30, n - 1, n, n + 9):
        got = qm.select_pages(q.to(dev), kv, ln.to(dev), table.to(dev), k, first=0)
        assert torch.equal(got.cpu(), K.chosen(q, cache, start, ln, table, k, 0, 1)), k


@pytest.mark.parametrize("new,HK,n", [([60, 40], 4, 700), ([900, 500], 1, 150), ([1, 1], 1, 2000)])
def test_work_groups_that_take_several_pages(qm, dev, new, HK, n):
    """More 64s of pages than work-groups of a token and key head: three, one, and all of them."""
    D, page = 32, 16
    lens = [n * page - 3, n * page // 3]
    cache = K.Cache(n + n // 3 + 4, HK, page, D, BF16, n, mean=True)
    start, ln, table, _ = K.batch(lens, new, page, cache.pages, n)
    q = queries(sum(new), 2 * HK, D, BF16, 5)
    kv = cache.on(qm, dev)
    got = qm.select_pages(q.to(dev), kv, ln.to(dev), table.to(dev), 9, start=start.to(dev))
    assert torch.equal(got.cpu(), K.chosen(q, cache, start, ln, table, 9, 1, 1))


def test_ties_and_special_scores(qm, dev):
    """Equal scores go to the lower page, zeros of either sign are one; scores that differ in their last bits are told apart; NaN and pages that
    are none come last, minus infinity among them, plus infinity first."""
    D, n = 64, 300
    cache = K.Cache(n, 1, 16, D, BF16, 0, mean=True)
    start, ln, table, _ = K.batch([16 * n], [1], 16, n, 0, spare=0)
    q = queries(1, 2, D, BF16, 1)
    for values in ("equal", "signs", "near", "special"):
        m = cache.mean
        if values == "equal":
            m[:] = m[0]
        elif values == "signs":
            m[:] = torch.where(torch.arange(n)[:, None, None] % 3 == 0, -0.0, 0.0).to(BF16)
        elif values == "near":  # (a sum of 64 products of which one is 2^-30 of the others)
            m[:] = 1.0
            m[:, 0, 5] = (torch.randperm(n, generator=torch.Generator().manual_seed(2)).float() * 2.0 ** -34).to(BF16)
            m[:, 0, 6] = 2.0 ** 10
        else:
            m[:] = torch.randn(m.shape, generator=torch.Generator().manual_seed(3)).to(BF16)
            for i, x in ((3, math.nan), (4, math.inf), (5, -math.inf)):
                m[i::7] = x
            table[0, 11] = -1
            table[0, 12] = n
        kv = cache.on(qm, dev)
        for k in (3, 100, 299):
            got = qm.select_pages(q.abs().to(dev), kv, ln.to(dev), table.to(dev), k)
            assert torch.equal(got.cpu(), K.chosen(q.abs(), cache, start, ln, table, k, 1, 1)), (values, k)


def test_rows_of_no_sequence_and_no_tokens(qm, dev):
    cache = K.Cache(30, 2, 16, 64, BF16, 0, mean=True)
    _, ln, table, _ = K.batch([100, 0, 200], [2, 1, 1], 16, 30, 0)
    start = torch.tensor([1, 3, 4, 5], dtype=torch.int32)
    q = queries(7, 4, 64, BF16, 1)
    kv = cache.on(qm, dev)
    sel = torch.full((7, 2, 4), 55, dtype=torch.int32, device=dev)
    qm.select_pages(q.to(dev), kv, ln.to(dev), table.to(dev), 4, start=start.to(dev), sel=sel)
    want = K.chosen(q, cache, start, ln, table, 4, 1, 1)
    live = torch.tensor([1, 2, 3, 4])
    assert torch.equal(sel.cpu()[live], want[live]) and bool((sel[[0, 5, 6]] == 55).all()) and bool((sel[3] == -1).all())


def test_graph(qm, dev):
    """Captured once; lengths are read at the replay."""
    cache = K.Cache(200, 2, 16, 64, BF16, 4, mean=True)
    start, ln, table, _ = K.batch([1500, 300, 20], [1, 1, 1], 16, 200, 4, spare=6)
    q = queries(3, 4, 64, BF16, 5)
    kv, qd, ld, td = cache.on(qm, dev), q.to(dev), ln.to(dev), table.to(dev)
    sel, ws = torch.empty((3, 2, 6), dtype=torch.int32, device=dev), qm.select_workspace(kv, 3, table.shape[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qm.select_pages(qd, kv, ld, td, 6, sel=sel, ws=ws)
    for step in range(3):
        graph.replay()
        eager = qm.select_pages(qd, kv, ld, td, 6)
        torch.cuda.synchronize()
        assert torch.equal(sel, eager) and torch.equal(sel.cpu(), K.chosen(q, cache, start, ld.cpu(), table, 6, 1, 1))
        ld.add_(14)


@pytest.mark.parametrize("ct", [BF16, E4M3])
def test_attention_layer_run(qm, dev, ct):
    """The operators as a layer uses them: a shared prompt and each sequence's own one appended, then decoding steps that append, attend over
    everything, choose pages and attend over those; every step against 64 bits on the cache as it is."""
    HQ, HK, D, page = 8, 2, 128, 16
    g = torch.Generator().manual_seed(6)
    kv = qm.KvCache.new(60, HK, page, D, ct, mean=True)
    f, w = inv_freq(D).to(dev), (torch.rand(D, generator=g) + 0.5).to(dev)
    prefix_len, lens = 290, [40, 3, 100]
    prefix = torch.arange(19, dtype=torch.int32)
    table = torch.full((3, 12), -1, dtype=torch.int32)
    perm = (torch.randperm(41, generator=g) + 19).tolist()
    for b in range(3):
        for j in range(9):
            table[b, j] = perm.pop()

    def append(T, slots, pos):
        x = torch.randn((T, (HQ + 2 * HK) * D), generator=g).to(BF16).to(dev)
        return qm.kv_append(x, HQ, kv, slots.to(torch.int32).to(dev), pos.to(torch.int32).to(dev), f, wq=w, wk=w, out=BF16)
    i = torch.arange(prefix_len)
    append(prefix_len, prefix[i // page] * page + i % page, i)
    place = lambda b, t: table[b, t // page] * page + t % page  # noqa: E731
    t = torch.cat([torch.arange(n) for n in lens])
    b = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
    q = append(len(t), place(b, t), t + prefix_len)
    start = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    ws = qm.attn_workspace(kv, 143, 3, HQ, prefix_len)
    ln = torch.tensor(lens, dtype=torch.int32)

    def held():
        c = K.Cache.__new__(K.Cache)
        c.pages, c.heads, c.page, c.D, c.dtype = 60, HK, page, D, ct
        c.data, c.scales, c.mean = [kv.k.cpu(), kv.v.cpu()], [None if s is None else s.cpu() for s in (kv.k_scale, kv.v_scale)], kv.mean.cpu()
        return c
    o = qm.attn_prefix(q, kv, ln.to(dev), table.to(dev), start=start.to(dev), prefix=prefix.to(dev), prefix_len=prefix_len, ws=ws)
    K.check(o, *K.attention(q.cpu(), held(), start, ln, table, BF16, None, prefix, prefix_len), BF16)
    one = torch.arange(4, dtype=torch.int32)
    for step in range(4):
        ln = ln + 1
        at = ln.long() - 1
        q = append(3, place(torch.arange(3), at), at + prefix_len)
        ld, td, c = ln.to(dev), table.to(dev), held()
        o = qm.attn_prefix(q, kv, ld, td, prefix=prefix.to(dev), prefix_len=prefix_len, ws=ws)
        K.check(o, *K.attention(q.cpu(), c, one, ln, table, BF16, None, prefix, prefix_len), BF16)
        sel = qm.select_pages(q, kv, ld, td, 4, last=2)
        assert torch.equal(sel.cpu(), K.chosen(q.cpu(), c, one, ln, table, 4, 1, 2))
        o = qm.attn_pages(q, kv, ld, td, sel, ws=ws)
        K.check(o, *K.attention(q.cpu(), c, one, ln, table, BF16, sel=sel.cpu()), BF16)
    a8, asc = qm.quantize_fp8(o.view(3, HQ * D))  # (what the next product takes)
    assert a8.shape == (3, HQ * D) and torch.isfinite(asc).all()
    vals = held().values()[0]
    for p in prefix[:18].tolist():
        assert bool(((kv.mean[p].cpu().double() - vals[p].mean(1)).abs() <= 20 * P.U32 * vals[p].abs().mean(1) + 1.01 * P.HALF[BF16] * vals[p].mean(1).abs()).all())
