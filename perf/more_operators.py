"""Performance cases of the paged cache of keys and values and of what reads it, through arcinfer_amd.qmatmul.

Kinds of case (a dict of plain values):
  append  QKV rows [q heads | k heads | v heads] of T tokens: RMS norm and rotation of the query and key heads, keys and values
          to the tokens' places in the cache (e4m3 with a scale for each token and head, or 16 bits), the mean of the keys of
          each page that becomes complete. Outputs: q and the cache
  attn    attention of each sequence's new tokens over `prefix` tokens that all sequences share and over the sequence's own
          ones up to the token itself. Output: o
  select  the k pages that each token's query heads score highest against the pages' mean keys, the first and the last two
          always among them. Output: the pages' numbers in the sequence, ascending, -1 behind them
  pages   attention over chosen pages only, for each token and key head others. Output: o

The sequences of a batch are `B`, their old tokens' counts spread evenly over the logarithm of lo..hi, the new ones' over 1..n.
Caches are [pages, key heads, page, D], a sequence's pages anywhere in them.
"""
import math

import torch

own = False

EPS = 1e-6
TOP = 448.0  # the largest e4m3 value
TINY = 2.0 ** -100  # heads whose largest value is below this are held as zeros
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
FIRST, LAST = 1, 2  # pages that are always among the chosen ones


def listed():
    return [
        # the smallest: four decoding tokens, heads of 256 of which a quarter turns
        {"name": "append_decode4", "kind": "append", "B": 4, "n": 1, "lo": 100, "hi": 3000, "HQ": 24, "HK": 4, "D": 256,
         "rot": 64, "pairs": "halves", "norm": True, "page": 64, "x": "f32", "q": "bf16", "cache": "bf16", "mean": False},
        # ragged prompts of a batch on small pages
        {"name": "append_ragged_16", "kind": "append", "B": 9, "n": 170, "lo": 7, "hi": 500, "HQ": 16, "HK": 16, "D": 80,
         "rot": 80, "pairs": "adjacent", "norm": False, "page": 16, "x": "f16", "q": "f16", "cache": "f16", "mean": False},
        # a long prompt into an 8-bit cache, with the pages' means for a later choice among them
        {"name": "append_prompt4096_e4m3", "kind": "append", "B": 1, "n": 4096, "lo": 30, "hi": 30, "HQ": 32, "HK": 8,
         "D": 128, "rot": 128, "pairs": "halves", "norm": True, "page": 64, "x": "bf16", "q": "bf16", "cache": "e4m3",
         "mean": True},
        # one decoding sequence of medium length, nothing shared
        {"name": "attn_decode1", "kind": "attn", "B": 1, "n": 1, "prefix": 0, "lo": 5000, "hi": 5000, "HQ": 24, "HK": 4,
         "D": 256, "page": 64, "cache": "bf16", "q": "bf16", "o": "bf16"},
        # a decoding batch behind one long system prompt
        {"name": "attn_prefix_batch48", "kind": "attn", "B": 48, "n": 1, "prefix": 8192, "lo": 16, "hi": 1500, "HQ": 32,
         "HK": 8, "D": 128, "page": 64, "cache": "bf16", "q": "bf16", "o": "bf16"},
        # questions on one very long document, 8-bit cache
        {"name": "attn_prefix_long_e4m3", "kind": "attn", "B": 16, "n": 1, "prefix": 65000, "lo": 50, "hi": 2000, "HQ": 32,
         "HK": 8, "D": 128, "page": 128, "cache": "e4m3", "q": "bf16", "o": "bf16"},
        # verification of up to five drafted tokens for a ragged batch, nothing shared
        {"name": "attn_verify5", "kind": "attn", "B": 12, "n": 5, "prefix": 0, "lo": 500, "hi": 20000, "HQ": 24, "HK": 4,
         "D": 256, "page": 32, "cache": "f16", "q": "f16", "o": "f16"},
        # chunks of prompts behind a shared prefix, f32 result for rows that are quantized next
        {"name": "attn_prompt3", "kind": "attn", "B": 3, "n": 1500, "prefix": 1000, "lo": 200, "hi": 2000, "HQ": 32, "HK": 8,
         "D": 128, "page": 16, "cache": "bf16", "q": "bf16", "o": "f32"},
        # one sequence of a long context
        {"name": "select_1", "kind": "select", "B": 1, "n": 1, "lo": 100000, "hi": 100000, "HQ": 24, "HK": 4, "D": 256,
         "page": 64, "k": 64, "q": "bf16"},
        # a decoding batch of long contexts
        {"name": "select_batch32", "kind": "select", "B": 32, "n": 1, "lo": 4000, "hi": 60000, "HQ": 32, "HK": 8, "D": 128,
         "page": 64, "k": 32, "q": "bf16"},
        # the same batch's attention over the chosen pages
        {"name": "pages_batch32", "kind": "pages", "B": 32, "n": 1, "lo": 4000, "hi": 20000, "HQ": 32, "HK": 8, "D": 128,
         "page": 64, "k": 32, "cache": "bf16", "q": "bf16", "o": "bf16"},
        # the tokens of a prompt's last chunk, each with pages of its own, 8-bit cache
        {"name": "pages_prompt_e4m3", "kind": "pages", "B": 2, "n": 150, "lo": 5000, "hi": 9000, "HQ": 24, "HK": 4, "D": 256,
         "page": 32, "k": 24, "cache": "e4m3", "q": "f16", "o": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attn", "attn", "attn", "select", "pages", "pages"))
    D = rng.choice((64, 80, 96, 128, 128, 192, 256))
    HK = rng.choice((1, 2, 4, 8))
    HQ = HK * rng.choice((1, 2, 4, 6, 8, 16))
    page = rng.choice((16, 32, 64, 64, 128, 256))
    cache = rng.choice(("bf16", "f16", "e4m3"))
    q = rng.choice(("bf16", "f16")) if cache == "e4m3" else cache
    c = {"kind": kind, "HQ": HQ, "HK": HK, "D": D, "page": page, "q": q}
    if kind == "append":
        c |= {"cache": cache, "mean": rng.random() < 0.5, "x": rng.choice(("f32", "bf16", "f16")), "norm": rng.random() < 0.75,
              "rot": rng.choice((D, D, D // 2, D // 4 * 2)), "pairs": rng.choice(("halves", "halves", "adjacent")),
              "B": _log_int(rng, 1, 64), "lo": _log_int(rng, 1, 1000)}
        T = _log_int(rng, 1, max(1, min(4096, 4096 * 40 * 128 // ((HQ + 2 * HK) * D))))
        c |= {"n": max(1, 2 * T // c["B"] - 1) if c["B"] > 1 else T, "hi": c["lo"] * rng.randint(1, 40)}
        return c
    if kind == "attn":
        c |= {"cache": cache, "o": rng.choice((q, q, "f32")), "B": _log_int(rng, 1, 64)}
        c["n"] = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 1500)))
        c["prefix"] = rng.choice((0, _log_int(rng, 1, 65536)))
        c["lo"] = _log_int(rng, 1, 2000)
        c["hi"] = _log_int(rng, c["lo"], 30000)
        # (within the largest listed case's work, and memory for the plain form's scores)
        while work(c)["flops"] > 7.4e10 or work(c)["bytes"] > 2.5e8 or _attn_rows(c) * HK * D > 3e8:
            c["B"], c["n"], c["prefix"] = (c["B"] + 1) // 2, (c["n"] + 1) // 2, c["prefix"] // 2
            c["hi"] = max(c["lo"], c["hi"] // 2)
        return c
    c |= {"B": _log_int(rng, 1, 48), "n": rng.choice((1, 1, 1, rng.randint(2, 200))), "lo": _log_int(rng, 1, 8000),
          "k": rng.choice((4, 8, 16, 32, 64, 100))}
    c["hi"] = c["lo"] * rng.randint(1, 12)
    if kind == "pages":
        c |= {"cache": cache, "o": rng.choice((q, q, "f32"))}
        while (work(c)["bytes"] > 2.5e8 or _attn_rows(c | {"prefix": 0}) * HK * D > 3e8
               or sum(_counts(c)[1]) * c["k"] * page * HK * D > 1e9):
            c["B"], c["n"], c["k"], c["hi"] = (c["B"] + 1) // 2, (c["n"] + 1) // 2, max(4, c["k"] // 2), max(c["lo"], c["hi"] // 2)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _counts(case):
    """Old and new tokens of each sequence, before they are put in the seed's order."""
    B, n, lo, hi = case["B"], case["n"], case["lo"], case["hi"]
    old = [int(round(lo * (hi / lo) ** ((i + 0.5) / B))) for i in range(B)]
    # (the i-th new count goes with the place (5 i) % B of the old ones, so that long and short ones meet)
    new = [n if B == 1 else 1 + (n - 1) * ((5 * i + 2) % B) // (B - 1) for i in range(B)]
    return old, new


def _visible(case):
    return sum(n * (case["prefix"] + o) + n * (n + 1) // 2 for o, n in zip(*_counts(case)))


def _attn_rows(case):
    """Tokens that the plain form gathers."""
    old, new = _counts(case)
    return case["prefix"] + case["B"] * (max(o + n for o, n in zip(old, new)) + case["page"])


def _batch(case, seed):
    """start [B + 1], lens [B] (new tokens among them), table [B, W] (-1 behind a sequence's pages), the prefix's pages, and how
    many pages there are."""
    old, new = _counts(case)
    order = torch.randperm(case["B"], generator=torch.Generator().manual_seed(seed)).tolist()
    old, new = [old[i] for i in order], [new[i] for i in order]
    P = case["page"]
    lens = torch.tensor([o + n for o, n in zip(old, new)])
    start = torch.tensor([0] + new).cumsum(0)
    n_pages = (lens + P - 1) // P
    shared = (case.get("prefix", 0) + P - 1) // P
    total = int(n_pages.sum()) + shared + 3
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    W = int(n_pages.max())
    j = torch.arange(W)
    at = (shared + n_pages.cumsum(0) - n_pages)[:, None] + j
    table = torch.where(j < n_pages[:, None], perm[at.clamp(max=total - 1)], -1)
    i32 = lambda t: t.to(torch.int32).cuda().contiguous()  # noqa: E731
    return {"start": i32(start), "lens": i32(lens), "table": i32(table), "prefix": i32(perm[:shared]), "pages": total,
            "T": int(start[-1]), "n_most": max(new)}


def _queries(case, T, seed):
    return (torch.randn((T, case["HQ"], case["D"]), generator=_gen(seed), device="cuda") * 1.5).to(DT[case["q"]])


def _cache_side(case, pages, seed, bias):
    """[pages, HK, page, D] of the cache's type, and the scales [pages, HK, page] of an 8-bit one. Keys have a part in common."""
    HK, P, D = case["HK"], case["page"], case["D"]
    x = torch.randn((pages, HK, P, D), generator=_gen(seed), device="cuda")
    if bias:
        x += torch.randn((HK, 1, D), generator=_gen(seed + 1), device="cuda")
    if case["cache"] != "e4m3":
        return x.to(DT[case["cache"]]), None
    sc = x.abs().amax(3) / TOP
    return x.div_(sc[..., None]).clamp_(-TOP, TOP).to(torch.float8_e4m3fn), sc


def _inv_freq(case):
    i = torch.arange(case["rot"] // 2, dtype=torch.float64)
    return (1e6 ** (-2.0 * i / max(1, case["rot"]))).float().cuda()


def _chosen(case, s, seed):
    """Pages for each token and key head, ascending, -1 behind them: the first, the last two, others at random."""
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["start"][1:], t.to(torch.int32), right=True)
    at = s["lens"][b] - (s["start"][b + 1] - t.to(torch.int32))  # the token's place in its sequence
    n = (at // case["page"] + 1)[:, None, None]
    W, k = s["table"].size(1), case["k"]
    j = torch.arange(max(W, k), device="cuda")
    r = torch.rand((s["T"], case["HK"], max(W, k)), generator=_gen(seed), device="cuda")
    r = torch.where((j < FIRST) | (j >= n - LAST), 2.0, r)
    r = torch.where(j < n, r, -1.0)
    pick = r.topk(k, 2).indices
    pick = torch.where(pick < n, pick, 2 ** 30).sort(2).values
    return torch.where(pick < 2 ** 30, pick, -1).to(torch.int32).contiguous()


def prepare(case, seed):
    seed = seed * 16
    s = {"case": case, **_batch(case, seed)}
    kind, T, HK, D = case["kind"], s["T"], case["HK"], case["D"]
    if kind == "append":
        g = _gen(seed + 2)
        s["x"] = (torch.randn((T, (case["HQ"] + 2 * HK) * D), generator=g, device="cuda") * 2.0).to(DT[case["x"]])
        s["wq"] = torch.rand(D, generator=g, device="cuda") + 0.5
        s["wk"] = torch.rand(D, generator=g, device="cuda") + 0.5
        s["inv_freq"] = _inv_freq(case)
        s |= _places(case, s)
    else:
        s["q"] = _queries(case, T, seed + 2)
    if kind == "select":  # (the keys themselves are not read)
        s["k"] = s["v"] = torch.empty((s["pages"], HK, case["page"], D), dtype=DT[case["q"]], device="cuda")
        s["k_scale"] = s["v_scale"] = None
    else:
        s["k"], s["k_scale"] = _cache_side(case, s["pages"], seed + 3, True)
        s["v"], s["v_scale"] = _cache_side(case, s["pages"], seed + 5, False)
    s["mean"] = None
    if kind == "select":
        s["mean"] = (torch.randn((s["pages"], HK, D), generator=_gen(seed + 7), device="cuda") * 0.2).to(torch.bfloat16)
    elif case.get("mean"):
        s["mean"] = torch.zeros((s["pages"], HK, D), dtype=torch.bfloat16, device="cuda")
    if kind == "pages":
        s["sel"] = _chosen(case, s, seed + 8)
    if own:  # a program keeps the cache's description and the workspace
        from arcinfer_amd import qmatmul as qm
        s["kv"] = qm.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["mean"])
        if kind == "attn":
            s["ws"] = qm.attn_workspace(s["kv"], T, case["B"], case["HQ"], case["prefix"])
        elif kind == "pages":
            s["ws"] = qm.attn_workspace(s["kv"], T, T, case["HQ"])
        elif kind == "select":
            s["ws"] = qm.select_workspace(s["kv"], T, s["table"].size(1))
    return s


def _places(case, s):
    """The positions and slots of the new tokens, as a scheduler keeps them for all layers, and the pages that they fill."""
    P = case["page"]
    t = torch.arange(s["T"], dtype=torch.int32, device="cuda")
    b = torch.searchsorted(s["start"][1:], t, right=True)
    pos = s["lens"][b] - (s["start"][b + 1] - t)
    slots = s["table"][b, (pos // P).long()] * P + pos % P
    last = slots[pos % P == P - 1]
    return {"pos": pos.contiguous(), "slots": slots.to(torch.int32).contiguous(), "full": (last // P).long()}


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _cache_out(s):
    return [t for t in (s["k"], s["v"], s["k_scale"], s["v_scale"], s["mean"]) if t is not None]


def _own(s):
    from arcinfer_amd import qmatmul as qm
    case = s["case"]
    start = None if case["n"] == 1 else s["start"]  # (one new token in each sequence needs no list)
    if case["kind"] == "append":
        norm = case["norm"]
        q = qm.kv_append(s["x"], case["HQ"], s["kv"], s["slots"], s["pos"], s["inv_freq"], wq=s["wq"] if norm else None,
                         wk=s["wk"] if norm else None, eps=EPS, adjacent=case["pairs"] == "adjacent", out=DT[case["q"]])
        return [q] + _cache_out(s)
    if case["kind"] == "attn":
        return qm.attn_prefix(s["q"], s["kv"], s["lens"], s["table"], start=start, prefix=s["prefix"],
                              prefix_len=case["prefix"], out=DT[case["o"]], ws=s["ws"])
    if case["kind"] == "select":
        return qm.select_pages(s["q"], s["kv"], s["lens"], s["table"], case["k"], start=start, first=FIRST, last=LAST, ws=s["ws"])
    return qm.attn_pages(s["q"], s["kv"], s["lens"], s["table"], s["sel"], start=start, out=DT[case["o"]], ws=s["ws"])


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _turned(x, w, cos, sin, case):
    """x [T, H, D] in 32 bits: normed by w where there is one, and turned."""
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w
    r = case["rot"]
    t = x[..., :r]
    u, v = (t[..., 0::2], t[..., 1::2]) if case["pairs"] == "adjacent" else (t[..., :r // 2], t[..., r // 2:])
    a, b = u * cos - v * sin, v * cos + u * sin
    t = torch.stack([a, b], -1).flatten(-2) if case["pairs"] == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([t, x[..., r:]], -1)


def _keep(cache, scales, page, at, x):
    """x [T, HK, D] in 32 bits to the places (page, at) of a cache [pages, HK, P, D]."""
    if scales is None:
        cache[page, :, at] = x.to(cache.dtype)
        return
    top = x.abs().amax(2)
    top = torch.where(top >= TINY, top, 0.0)
    x = x * torch.where(top > 0, TOP / top, 0.0)[..., None]
    cache.view(torch.uint8)[page, :, at] = x.to(cache.dtype).view(torch.uint8)
    scales[page, :, at] = top / TOP


def _plain_append(s):
    case = s["case"]
    T, D, HQ, HK, P = s["T"], case["D"], case["HQ"], case["HK"], case["page"]
    # (32 bits lose far positions)
    angle = (s["pos"].double()[:, None] * s["inv_freq"].double())[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = s["x"].view(T, HQ + 2 * HK, D).float()
    q = _turned(x[:, :HQ], s["wq"], cos, sin, case).to(DT[case["q"]])
    page, at = (s["slots"] // P).long(), (s["slots"] % P).long()
    _keep(s["k"], s["k_scale"], page, at, _turned(x[:, HQ:HQ + HK], s["wk"], cos, sin, case))
    _keep(s["v"], s["v_scale"], page, at, x[:, HQ + HK:])
    if s["mean"] is not None:
        k = s["k"].view(torch.uint8)[s["full"]].view(s["k"].dtype) if s["k_scale"] is not None else s["k"][s["full"]]
        k = k.float() if s["k_scale"] is None else k.float() * s["k_scale"][s["full"]][..., None]
        s["mean"][s["full"]] = k.mean(2).to(torch.bfloat16)
    return [q] + _cache_out(s)


def _gathered(cache, scales, pages):
    """The rows of `pages` [..., n] in 32 bits: [..., HK, n * P, D]."""
    c = cache.view(torch.uint8)[pages].view(cache.dtype) if scales is not None else cache[pages]
    c = c.float() if scales is None else c.float() * scales[pages][..., None]
    c = c.movedim(-3, -4)  # [..., HK, n, P, D]
    return c.reshape(*c.shape[:-3], c.shape[-3] * c.shape[-2], c.shape[-1])


def _rows_of(s, t):
    """Rows [T, ...] as [B, n_most, ...], the rest zeros, and the index that takes them back."""
    B, n = s["case"]["B"], s["n_most"]
    i = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["start"][1:], i.to(torch.int32), right=True)
    j = i - s["start"][b]
    r = torch.zeros((B, n) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda")
    r[b, j] = t
    return r, (b, j)


def _plain_attn(s):
    case = s["case"]
    T, B, D, HQ, HK, n = s["T"], case["B"], case["D"], case["HQ"], case["HK"], s["n_most"]
    G, scale = HQ // HK, D ** -0.5
    q = s["q"].float() * scale
    pages = s["table"].clamp(min=0).long()
    k, v = _gathered(s["k"], s["k_scale"], pages), _gathered(s["v"], s["v_scale"], pages)  # [B, HK, L, D]
    qb, back = _rows_of(s, q)
    qb = qb.view(B, n, HK, G, D).permute(0, 2, 1, 3, 4).reshape(B, HK, n * G, D)
    x = (qb @ k.transpose(2, 3).contiguous()).view(B, HK, n, G, -1)
    j = torch.arange(k.size(2), device="cuda")
    new = s["start"][1:] - s["start"][:-1]
    sees = s["lens"][:, None] - new[:, None] + torch.arange(n, device="cuda") + 1  # [B, n]
    # (what lies behind a sequence's own tokens is masked, and zeroed: it may hold anything)
    x = x.masked_fill((j >= sees[..., None])[:, None, :, None, :], float("-inf"))
    v = v.masked_fill((j >= s["lens"][:, None])[:, None, :, None], 0.0)
    top = x.amax(-1)
    if case["prefix"]:
        pk, pv = (_gathered(c, sc, s["prefix"].long())[:, :case["prefix"]] for c, sc in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        px = q.view(T, HK, G * D).transpose(0, 1).reshape(HK, T * G, D) @ pk.transpose(1, 2).contiguous()  # [HK, T G, Lp]
        ptop, _ = _rows_of(s, px.amax(-1).view(HK, T, G).transpose(0, 1))  # [B, n, HK, G]
        top = torch.maximum(top, ptop.permute(0, 2, 1, 3))
    e = torch.exp(x - top[..., None])
    total = e.sum(-1)
    o = e.view(B, HK, n * G, -1) @ v
    o = o.view(B, HK, n, G, D).permute(0, 2, 1, 3, 4)[back]  # [T, HK, G, D]
    total = total.permute(0, 2, 1, 3)[back]
    if case["prefix"]:
        e = torch.exp(px - top.permute(0, 2, 1, 3)[back].transpose(0, 1).reshape(HK, T * G, 1))
        total = total + e.sum(-1).view(HK, T, G).transpose(0, 1)
        o = o + (e @ pv).view(HK, T, G, D).transpose(0, 1)
    return (o / total[..., None]).reshape(T, HQ, D).to(DT[case["o"]])


def _plain_select(s):
    case = s["case"]
    T, B, D, HK, n = s["T"], case["B"], case["D"], case["HK"], s["n_most"]
    G, W, k = case["HQ"] // HK, s["table"].size(1), case["k"]
    # (64 bits: pages are chosen by which score is the larger, however near they are)
    mean = s["mean"][s["table"].clamp(min=0).long()].double().transpose(1, 2).contiguous()  # [B, HK, W, D]
    qb, back = _rows_of(s, s["q"].double())
    qb = qb.view(B, n, HK, G, D).permute(0, 2, 1, 3, 4).reshape(B, HK, n * G, D)
    x = (qb @ mean.transpose(2, 3).contiguous()).view(B, HK, n, G, W).amax(3).transpose(1, 2)[back]  # [T, HK, W]
    new = s["start"][1:] - s["start"][:-1]
    at = (s["lens"][:, None] - new[:, None] + torch.arange(n, device="cuda"))[back]
    pages = (at // case["page"] + 1)[:, None, None]
    j = torch.arange(W, device="cuda")
    x = x.masked_fill((j < FIRST) | (j >= pages - LAST), float("inf")).masked_fill(j >= pages, float("-inf"))
    pick = x.sort(dim=2, descending=True, stable=True).indices[..., :k]
    if k > W:
        pick = torch.cat([pick, pick.new_full((T, HK, k - W), W)], 2)
    pick = torch.where(pick < pages, pick, 2 ** 30).sort(2).values
    return torch.where(pick < 2 ** 30, pick, -1).to(torch.int32)


def _plain_pages(s):
    case = s["case"]
    T, D, HQ, HK, P = s["T"], case["D"], case["HQ"], case["HK"], case["page"]
    G = HQ // HK
    t = torch.arange(T, dtype=torch.int32, device="cuda")
    b = torch.searchsorted(s["start"][1:], t, right=True)
    at = s["lens"][b] - (s["start"][b + 1] - t)
    sel = s["sel"].long()
    page = torch.where(sel >= 0, s["table"][b[:, None, None], sel.clamp(min=0)].long(), 0)
    h = torch.arange(HK, device="cuda")[None, :, None]

    def rows(c, sc):
        r = c.view(torch.uint8)[page, h].view(c.dtype) if sc is not None else c[page, h]  # [T, HK, k, P, D]
        r = r.float() if sc is None else r.float() * sc[page, h][..., None]
        return r.reshape(T, HK, -1, D)
    place = (sel[..., None] * P + torch.arange(P, device="cuda")).view(T, HK, -1)
    seen = (place <= at[:, None, None]) & (sel >= 0).repeat_interleave(P, 2)
    x = (s["q"].float() * D ** -0.5).view(T, HK, G, D) @ rows(s["k"], s["k_scale"]).transpose(2, 3).contiguous()
    x = x.masked_fill(~seen[:, :, None], float("-inf"))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = e @ rows(s["v"], s["v_scale"]).masked_fill(~seen[..., None], 0.0)
    return (o / e.sum(-1, keepdim=True)).reshape(T, HQ, D).to(DT[case["o"]])


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attn": _plain_attn, "select": _plain_select, "pages": _plain_pages}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    old, new = _counts(case)
    T, HQ, HK, D, P, kind = sum(new), case["HQ"], case["HK"], case["D"], case["page"], case["kind"]
    q = T * HQ * D * SIZE[case["q"]]
    if kind == "append":
        b = T * (HQ + 2 * HK) * D * SIZE[case["x"]] + q + 2 * T * HK * (D * SIZE[case["cache"]] + (4 if case["cache"] == "e4m3" else 0))
        f = (4.0 * D + 3.0 * case["rot"]) * T * (HQ + HK)
        if case["mean"]:
            b += T // P * HK * D * 2
        return {"bytes": b + 8 * T, "flops": f}
    if kind == "select":
        pages = [(o + n + P - 1) // P for o, n in zip(old, new)]
        return {"bytes": sum(pages) * HK * D * 2 + q + 4 * T * HK * case["k"],
                "flops": 2.0 * HQ * D * sum(p * n for p, n in zip(pages, new))}
    token = 2 * HK * (D * SIZE[case["cache"]] + (4 if case["cache"] == "e4m3" else 0))
    o = T * HQ * D * SIZE[case["o"]]
    if kind == "attn":
        return {"bytes": (case["prefix"] + sum(old) + T) * token + q + o, "flops": 4.0 * HQ * D * _visible(case)}
    # (each page once for a sequence, however many of its tokens choose it)
    seen = [min(case["k"], (a + P) // P) * P for a, n in zip(old, new)]
    read = [min(a + n, s * n) for a, n, s in zip(old, new, seen)]
    return {"bytes": sum(read) * token + q + o + 4 * T * HK * case["k"], "flops": 4.0 * HQ * D * sum(s * n for s, n in zip(seen, new))}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------
def _wide(cache, scales):
    c = cache.float().double()
    return c if scales is None else c * scales.double()[..., None]


def _exact_append(case, seed, m):
    g = _gen(seed + 2)
    T, D, HQ, HK, P, rot = m["T"], case["D"], case["HQ"], case["HK"], case["page"], case["rot"]
    x = (torch.randn((T, (HQ + 2 * HK) * D), generator=g, device="cuda") * 2.0).to(DT[case["x"]]).double().view(T, -1, D)
    ws = [(torch.rand(D, generator=g, device="cuda") + 0.5).double() for _ in range(2)]
    f, half = _inv_freq(case).double(), rot // 2
    starts, lens, table = m["start"].tolist(), m["lens"].tolist(), m["table"].tolist()
    place = []  # (position, page) of each token
    for b, n in enumerate(lens):
        new = starts[b + 1] - starts[b]
        place += [(p, table[b][p // P]) for p in range(n - new, n)]
    pos = torch.tensor([p for p, _ in place], dtype=torch.float64, device="cuda")
    page = torch.tensor([p for _, p in place], device="cuda")
    at = pos.long() % P
    done = []
    for h0, h1, w in ((0, HQ, ws[0]), (HQ, HQ + HK, ws[1])):
        z = x[:, h0:h1].clone()
        if case["norm"]:
            z = z * w / torch.sqrt(z.pow(2).sum(2, keepdim=True) / D + EPS)
        y = z.clone()
        for i in range(half):  # each pair as one complex number, times e^(i angle)
            lo, hi = (2 * i, 2 * i + 1) if case["pairs"] == "adjacent" else (i, i + half)
            c = torch.complex(z[:, :, lo], z[:, :, hi]) * torch.polar(torch.ones_like(pos), pos * f[i])[:, None]
            y[:, :, lo], y[:, :, hi] = c.real, c.imag
        done.append(y)
    out, scales, held = [done[0]], [], None
    for c, y in ((_cache_side(case, m["pages"], seed + 3, True), done[1]), (_cache_side(case, m["pages"], seed + 5, False), x[:, HQ + HK:])):
        z = c[0].float().double()
        if c[1] is None:
            z[page, :, at] = y
            stored = c[0].float().double()
            stored[page, :, at] = y.to(c[0].dtype).double()
        else:
            top, sc = y.abs().amax(2), c[1].double()
            z[page, :, at] = y * (TOP / top)[..., None]
            sc[page, :, at] = top / TOP
            scales.append(sc)
            stored = z.float().to(torch.float8_e4m3fn).double() * sc[..., None]
        out.append(z)
        held = stored if held is None else held
    out += scales
    if case["mean"]:
        mean = torch.zeros((m["pages"], HK, D), dtype=torch.float64, device="cuda")
        for i, (p, g_) in enumerate(place):
            if p % P == P - 1:
                mean[g_] = held[g_].sum(1) / P
        out.append(mean)
    return out


def _exact_rows(case, m, seed):
    k = _wide(*_cache_side(case, m["pages"], seed + 3, True))
    v = _wide(*_cache_side(case, m["pages"], seed + 5, False))
    return k, v, _queries(case, m["T"], seed + 2).double()


def _exact_attn(case, seed, m):
    k, v, q = _exact_rows(case, m, seed)
    D, HK, P, Lp = case["D"], case["HK"], case["page"], case["prefix"]
    G = case["HQ"] // HK
    o = torch.zeros_like(q)
    starts, lens = m["start"].tolist(), m["lens"].tolist()
    for h in range(HK):
        pk, pv = (c[m["prefix"].long(), h].reshape(-1, D)[:Lp] for c in (k, v))
        for b, L in enumerate(lens):
            mine = m["table"][b, :(L + P - 1) // P].long()
            kk = torch.cat([pk, k[mine, h].reshape(-1, D)[:L]])
            vv = torch.cat([pv, v[mine, h].reshape(-1, D)[:L]])
            n = starts[b + 1] - starts[b]
            sees = Lp + L - n + torch.arange(n, device="cuda")[:, None]
            hidden = torch.arange(Lp + L, device="cuda") > sees
            for g in range(G):
                x = q[starts[b]:starts[b + 1], h * G + g] @ kk.t().contiguous() / math.sqrt(D)
                w = torch.softmax(x.masked_fill(hidden, float("-inf")), 1)
                o[starts[b]:starts[b + 1], h * G + g] = w @ vv
    return o


def _exact_select(case, seed, m):
    HK, D, P, k = case["HK"], case["D"], case["page"], case["k"]
    G = case["HQ"] // HK
    mean = (torch.randn((m["pages"], HK, D), generator=_gen(seed + 7), device="cuda") * 0.2).to(torch.bfloat16).double()
    q = _queries(case, m["T"], seed + 2).double()
    starts, lens = m["start"].tolist(), m["lens"].tolist()
    sel = torch.full((m["T"], HK, k), -1, dtype=torch.int32)
    for b, L in enumerate(lens):
        mine = mean[m["table"][b, :(L + P - 1) // P].long()]
        for t in range(starts[b], starts[b + 1]):
            n = (L - (starts[b + 1] - t)) // P + 1
            score = (mine[:n, :, None, :] * q[t].view(1, HK, G, D)).sum(3).max(2).values.cpu()  # [n, HK]
            for h in range(HK):
                must = {j for j in range(n) if j < FIRST or j >= n - LAST}
                free = sorted((j for j in range(n) if j not in must), key=lambda j: (-score[j, h].item(), j))
                pick = sorted((sorted(must) + free)[:k])
                sel[t, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return sel.cuda()


def _exact_pages(case, seed, m):
    k, v, q = _exact_rows(case, m, seed)
    D, HK, P = case["D"], case["HK"], case["page"]
    G = case["HQ"] // HK
    sel = _chosen(case, m, seed + 8).cpu()
    o = torch.zeros_like(q)
    starts, lens = m["start"].tolist(), m["lens"].tolist()
    for b, L in enumerate(lens):
        for t in range(starts[b], starts[b + 1]):
            last = L - (starts[b + 1] - t)
            for h in range(HK):
                pick = sel[t, h][sel[t, h] >= 0].cuda()
                pages = m["table"][b, pick.long()].long()
                here = ((pick[:, None] * P + torch.arange(P, device="cuda")) <= last).view(-1)
                kk, vv = (c[pages, h].reshape(-1, D)[here] for c in (k, v))
                w = torch.softmax(q[t, h * G:(h + 1) * G] @ kk.t().contiguous() / math.sqrt(D), 1)
                o[t, h * G:(h + 1) * G] = w @ vv
    return o


def exact(case, seed):
    seed = seed * 16
    m = _batch(case, seed)
    # (these two go token by token: long prompts would take minutes)
    if case["kind"] == "select" and m["T"] * case["HK"] * int(m["lens"].max()) // case["page"] > 1_500_000:
        return None
    if case["kind"] == "pages" and m["T"] * case["HK"] > 6000:
        return None
    return {"append": _exact_append, "attn": _exact_attn, "select": _exact_select, "pages": _exact_pages}[case["kind"]](case, seed, m)
