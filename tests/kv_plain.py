"""Plain 64-bit forms of the paged cache's operators, on the CPU: caches, attention with its error bound, the choice of pages."""
import math

import torch

from tests import fp8_plain as P

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


class Cache:
    """A cache on the CPU, [pages, heads, page, D] of `dtype`, and its values in 64 bits."""

    def __init__(self, pages, heads, page, D, dtype, seed, mean=False):
        g = torch.Generator().manual_seed(seed)
        x = [torch.randn((pages, heads, page, D), generator=g) for _ in range(2)]
        x[0] += torch.randn((1, heads, 1, D), generator=g)
        self.scales = [None, None]
        if dtype == E4M3:
            self.scales = [t.abs().amax(3) / P.TOP for t in x]
            x = [t / s[..., None] for t, s in zip(x, self.scales)]
        self.data = [t.to(dtype) for t in x]
        self.mean = (torch.randn((pages, heads, D), generator=g) * 0.3).to(BF16) if mean else None
        self.pages, self.heads, self.page, self.D, self.dtype = pages, heads, page, D, dtype

    def values(self):
        v = [t.float().double() for t in self.data]
        return [a if s is None else a * s.double()[..., None] for a, s in zip(v, self.scales)]

    def on(self, qm, dev, order=(0, 1, 2), pad=0):
        """A KvCache of copies on the GPU, its dimensions lying in `order` (the outermost first), `pad` elements behind each row."""
        put = lambda t: None if t is None else t.to(dev)  # noqa: E731

        def laid(t):
            raw = t.view(torch.uint8) if t.dtype == E4M3 else t
            n = [raw.shape[i] for i in order]
            buf = torch.full((*n, self.D + pad), 77, dtype=raw.dtype, device=dev)
            view = buf[..., :self.D].permute(*[order.index(i) for i in range(3)], 3)
            view.copy_(raw)
            return view.view(t.dtype)
        return qm.KvCache(laid(self.data[0]), laid(self.data[1]), put(self.scales[0]), put(self.scales[1]), put(self.mean))


def batch(lens, new, page, pages, seed, spare=2):
    """(start, lens, table) int32, page numbers of the sequences anywhere in 0 .. pages - 1, none of them twice."""
    need = [(n + page - 1) // page for n in lens]
    W = max(need + [1]) + spare
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(perm[:n], dtype=torch.int32)
        perm = perm[n:]
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    return start, torch.tensor(lens, dtype=torch.int32), table, perm


def rows_of(cache, h, pages, n):
    """Keys and values of the first n tokens in `pages` for key head h, and which of them are there."""
    P_ = cache.page
    k, v, there = [], [], []
    for i in range((n + P_ - 1) // P_):
        p = int(pages[i]) if i < len(pages) else -1
        ok = 0 <= p < cache.pages
        a, b = cache.vals
        k.append(a[p, h] if ok else torch.zeros((P_, cache.D), dtype=torch.float64))
        v.append(b[p, h] if ok else torch.zeros((P_, cache.D), dtype=torch.float64))
        there += [ok] * P_
    if not k:
        return (torch.zeros((0, cache.D), dtype=torch.float64),) * 2 + (torch.zeros(0, dtype=torch.bool),)
    return torch.cat(k)[:n], torch.cat(v)[:n], torch.tensor(there[:n])


def row(q, k, v, scale, dtype, out):
    """One row over the keys that it sees: the result, and how far a sum in f32 may be off."""
    L, D = k.shape
    if L == 0:
        return torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    x = (k @ q) * scale
    p = torch.softmax(x, 0)
    o = p @ v
    U = P.U32
    # the logit: D exact products added on the matrix pipe (an addition may lose a whole step), the scale's, log2 e's and an 8-bit key's scale's
    # roundings, the difference to the maximum; then the exponential's 2 steps and an 8-bit value's scale
    e = 2 * D * U * (k.abs() @ q.abs()) * abs(scale) + 5 * U * x.abs() + U * (x - x.max()).abs() + 6 * U
    # the weight's rounding for the second product: by parts of the matrix pipe's type
    pipe = F16 if dtype == F16 else BF16
    parts = 1 if (out == BF16 or (out == F16 and dtype == F16)) else 2
    half = P.HALF[pipe] ** parts
    # f16 weights below 2^-14 of 2^6 times the largest: half a step of 2^-24 against 2^6
    floor = 2.0 ** -31 if pipe == F16 else 0.0
    # L products added, and the sum of L weights; rescaling when a maximum is renewed, joining waves and pieces
    bound = (p * (e + half)) @ v.abs() + (3 * L + 100) * U * (p @ v.abs()) + ((p * e).sum() + L * U) * o.abs() + floor * v.abs().sum(0)
    return o, bound


def attention(q, cache, start, lens, table, out, scale=None, prefix=(), prefix_len=0, sel=None):
    """(o, bound) [T, HQ, D] in 64 bits; rows of no sequence are NaN in o."""
    T, HQ, D = q.shape
    G = HQ // cache.heads
    scale = D ** -0.5 if scale is None else scale
    cache.vals = cache.values()
    o = torch.full((T, HQ, D), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(o)
    q = q.double()
    for b in range(len(lens)):
        t0, t1 = int(start[b]), int(start[b + 1])
        for t in range(t0, t1):
            see = max(0, min(int(lens[b]) - (t1 - t) + 1, table.shape[1] * cache.page))
            for h in range(cache.heads):
                if sel is None:
                    pk, pv, pt = rows_of(cache, h, prefix, prefix_len)
                    k, v, there = rows_of(cache, h, table[b], see)
                    k, v = torch.cat([pk[pt], k[there]]), torch.cat([pv[pt], v[there]])
                else:
                    ks, vs = [], []
                    for j in sel[t, h].tolist():
                        if 0 <= j < table.shape[1] and 0 <= int(table[b, j]) < cache.pages:
                            n = max(0, min(cache.page, see - j * cache.page))
                            ks.append(cache.vals[0][int(table[b, j]), h, :n])
                            vs.append(cache.vals[1][int(table[b, j]), h, :n])
                    k = torch.cat(ks) if ks else torch.zeros((0, D), dtype=torch.float64)
                    v = torch.cat(vs) if vs else torch.zeros((0, D), dtype=torch.float64)
                for g in range(G):
                    o[t, h * G + g], bound[t, h * G + g] = row(q[t, h * G + g], k, v, scale, cache.dtype, out)
    return o, bound


def check(got, o, bound, out):
    live = ~torch.isnan(o).all(2)
    off = (got.double().cpu() - o).abs()[live]
    allowed = (bound + P.rounding(out, o) + 1e-40)[live]
    assert bool((off <= allowed).all()), float((off / allowed).max())


def chosen(q, cache, start, lens, table, k, first, last):
    """The pages of qmatmul_select_pages; rows of no sequence -1."""
    T, HQ, D = q.shape
    G, P_ = HQ // cache.heads, cache.page
    sel = torch.full((T, cache.heads, k), -1, dtype=torch.int32)
    q, mean = q.double(), cache.mean.double()
    for b in range(len(lens)):
        t0, t1 = int(start[b]), int(start[b + 1])
        for t in range(t0, t1):
            at = int(lens[b]) - (t1 - t)
            n = min(at // P_ + 1, table.shape[1]) if at >= 0 else 0
            for h in range(cache.heads):
                if n <= k:
                    sel[t, h, :n] = torch.arange(n, dtype=torch.int32)
                    continue
                score = []
                for j in range(n):
                    p = int(table[b, j])
                    s = (q[t, h * G:(h + 1) * G] * mean[p, h]).sum(1) if 0 <= p < cache.pages else torch.tensor([math.nan])
                    s = s[~torch.isnan(s)]
                    score.append(float(s.max()) if len(s) else -math.inf)
                must = [j for j in range(n) if j < first or j >= n - last]
                free = sorted((j for j in range(n) if j not in must), key=lambda j: (-score[j], j))
                sel[t, h] = torch.tensor(sorted((must + free)[:k]), dtype=torch.int32)
    return sel
