"""Appending to a paged cache on the GPU against its 64-bit form (tests/fp8_plain.py, tests/kv_plain.py)."""
import numpy as np
import pytest
import torch

from tests import fp8_plain as P
from tests import kv_plain as K

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def inv_freq(rot, theta=1e6):
    i = np.arange(rot // 2, dtype=np.float64)
    return torch.from_numpy((theta ** (-2.0 * i / max(1, rot))).astype(np.float32))


def turned(x, w, pos, f, adjacent, sections=None, turns=False, scale=1.0, seq=16):
    """[T, H, D] in 64 bits and how far f32 may be off: the norm, and the rotation as tests/test_gpu_qk_norm_rope.py counts it."""
    y, B = P.rotated(x.double(), None if w is None else w.double(), 1e-6, pos, f, sections or [len(f)], turns, adjacent, scale)
    return y, ((P.norm_error(x.shape[2], seq) if w is not None else 0) + (4 + np.pi + 2 + 1 + 3) * P.U32) * B + 1e-40


def stored(cache, scales, y, err, slots, page, before, before_scales):
    """The cache against rows y [T, H, D] known up to err; every other place as it was."""
    now = cache.cpu()
    live = (slots >= 0) & (slots < now.shape[0] * page)
    pg, at = (slots[live] // page).long(), (slots[live] % page).long()
    y, err = y[live], err[live]
    if scales is None:
        got = now[pg, :, at].double()
        assert bool(((got - y).abs() <= err + P.rounding(now.dtype, y)).all())
    else:
        sc = scales.cpu()
        top = y.abs().amax(2)
        top = torch.where(top >= P.TINY, top, torch.zeros_like(top))
        # the scale: the largest value, off by what it is known up to, and the quotient's rounding
        assert bool(((sc[pg, :, at].double() - top / P.TOP).abs() <= err.amax(2) / P.TOP + P.U32 * top).all())
        # the values over the scale, 448 / amax rounded and the product too
        safe = torch.where(top > 0, top, torch.ones_like(top))[..., None]
        q, e = y / safe * P.TOP, (err + err.amax(2, keepdim=True) * (y / safe).abs()) / safe * P.TOP + 3 * P.U32 * 448
        q, e = torch.where(top[..., None] > 0, q, 0.0), torch.where(top[..., None] > 0, e, 0.0)
        assert P.near_e4m3(P.value(now.view(torch.uint8)[pg, :, at]), q, e)
        sc2, b2 = sc.clone(), before_scales.clone()
        sc2[pg, :, at] = 0
        b2[pg, :, at] = 0
        assert torch.equal(sc2, b2)
    raw = lambda t: t.view(torch.uint8 if t.dtype == E4M3 else torch.int16).clone()  # noqa: E731
    a, b = raw(now), raw(before)
    a[pg, :, at] = 0
    b[pg, :, at] = 0
    assert torch.equal(a, b)


def run(qm, dev, T, HQ, HK, D, rot, page, xt, qt, ct, adjacent=False, norm=True, seed=0, mean=False, order=(0, 1, 2), pad=0, off=0, pages=None):
    g = torch.Generator().manual_seed(seed)
    pages = pages or (T + page - 1) // page + 2
    cache = K.Cache(pages, HK, page, D, ct, seed, mean)
    kv = cache.on(qm, dev, order, pad)
    x = torch.randn((T, (HQ + 2 * HK) * D + 2 * off), generator=g).mul_(3).to(xt)
    wq, wk = torch.rand(D, generator=g) + 0.5, torch.rand(D, generator=g) + 0.5
    pos = torch.randint(0, 300000, (T,), generator=g, dtype=torch.int32)
    f = inv_freq(rot)
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    w = dict(wq=wq.to(dev), wk=wk.to(dev)) if norm else {}
    q = qm.kv_append(x.to(dev), HQ, kv, slots.to(dev), pos.to(dev), f.to(dev), adjacent=adjacent, out=qt, q_off=off, **w)
    assert q.shape == (T, HQ, D) and q.dtype == qt
    xs = x[:, off:off + (HQ + 2 * HK) * D].reshape(T, -1, D)
    y, e = turned(xs[:, :HQ], wq if norm else None, pos[None], f, adjacent)
    assert bool(((q.double().cpu() - y).abs() <= e + P.rounding(qt, y)).all())
    y, e = turned(xs[:, HQ:HQ + HK], wk if norm else None, pos[None], f, adjacent)
    stored(kv.k, kv.k_scale, y, e, slots, page, cache.data[0], cache.scales[0])
    v = xs[:, HQ + HK:].double()
    stored(kv.v, kv.v_scale, v, torch.zeros_like(v), slots, page, cache.data[1], cache.scales[1])
    if mean:
        vals = kv.k.cpu().float().double() if ct != E4M3 else P.value(kv.k.cpu().view(torch.uint8)) * kv.k_scale.cpu().double()[..., None]
        want, full = cache.mean.double().clone(), (slots[slots % page == page - 1] // page).long()
        want[full] = vals[full].mean(2)
        # page sums in f32 (an 8-bit key's product is within the fma), the quotient, rounded to bf16
        bound = torch.zeros_like(want)
        bound[full] = (page + 2) * P.U32 * vals[full].abs().mean(2) + P.HALF[BF16] * want[full].abs() * 1.01
        assert bool(((kv.mean.cpu().double() - want).abs() <= bound).all())
    return kv, slots


SHAPES = [(1, 1, 1, 16, 16, 16), (3, 8, 2, 128, 128, 64), (5, 24, 4, 256, 64, 64), (7, 4, 4, 80, 80, 16), (33, 5, 1, 96, 48, 32),
          (130, 6, 3, 64, 30, 128), (9, 2, 1, 144, 0, 256), (1100, 4, 2, 64, 64, 16), (17, 0, 3, 32, 32, 16)]


@pytest.mark.parametrize("xt,qt", [(F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("ct", [BF16, F16, E4M3])
@pytest.mark.parametrize("T,HQ,HK,D,rot,page", SHAPES)
def test_shapes_and_types(qm, dev, T, HQ, HK, D, rot, page, ct, xt, qt):
    for adjacent in (False, True):
        run(qm, dev, T, HQ, HK, D, rot, page, xt, qt, ct, adjacent, norm=adjacent == (T % 2 == 1), seed=T + D)


@pytest.mark.parametrize("ct", [BF16, F16, E4M3])
@pytest.mark.parametrize("D,page", [(64, 16), (80, 32), (256, 64), (128, 256)])
def test_means_of_filled_pages(qm, dev, D, page, ct):
    """Scattered tokens fill pages among which others stay as they are."""
    _, slots = run(qm, dev, 6 * page, 2, 2, D, D, page, F32, BF16, ct, mean=True, seed=D, pages=6)
    assert int((slots % page == page - 1).sum()) == 6
    run(qm, dev, 3 * page, 2, 3, D, D, page, BF16, BF16, ct, mean=True, seed=D, pages=4)


@pytest.mark.parametrize("ct", [F16, E4M3])
@pytest.mark.parametrize("order,pad", [((0, 2, 1), 0), ((1, 0, 2), 0), ((0, 1, 2), 16), ((2, 1, 0), 32)])
def test_cache_strides(qm, dev, order, pad, ct):
    run(qm, dev, 40, 4, 2, 80, 80, 32, BF16, BF16, ct, order=order, pad=pad, mean=True, pages=2)


@pytest.mark.parametrize("off", [1, 3, 4])
@pytest.mark.parametrize("xt", [F32, F16])
def test_rows_of_any_alignment(qm, dev, off, xt):
    for ct in (BF16, E4M3):
        run(qm, dev, 21, 3, 2, 64, 64, 16, xt, F16, ct, off=off)
        run(qm, dev, 21, 3, 2, 256, 64, 16, xt, F16, ct, off=off)


def test_as_the_rotation_does_it(qm, dev):
    """Queries and 16-bit keys have the bits of qk_norm_rope, several axes among them; values are the rows' own."""
    T, HQ, HK, D = 50, 6, 2, 128
    g = torch.Generator().manual_seed(1)
    x = torch.randn((T, (HQ + 2 * HK) * D), generator=g).to(BF16).to(dev)
    w = (torch.rand(D, generator=g) + 0.5).to(dev)
    slots = torch.randperm(64, generator=g)[:T].to(torch.int32).to(dev)
    for pos, sections, turns in ((torch.arange(T, dtype=torch.int32), None, False), (torch.randint(0, 999, (3, T), generator=g, dtype=torch.int32), (16, 8, 8), True)):
        f = inv_freq(64).to(dev)
        for ct in (BF16, F16):
            kv = qm.KvCache.new(4, HK, 16, D, ct)
            got = qm.kv_append(x, HQ, kv, slots, pos.to(dev), f, wq=w, wk=w, sections=sections, turns=turns, scale=1.5, out=ct)
            q, k = qm.qk_norm_rope(x, HQ, HK, D, pos.to(dev), f, wq=w, wk=w, sections=sections, turns=turns, scale=1.5, out=ct)
            pg, at = (slots // 16).long(), (slots % 16).long()
            assert torch.equal(got, q) and torch.equal(kv.k[pg, :, at], k)
            assert torch.equal(kv.v[pg, :, at], x[:, (HQ + HK) * D:].view(T, HK, D).to(ct))


def test_head_offsets_and_in_place(qm, dev):
    """Heads apart from each other and values in front of the keys; q where it lies; keys and values in turns in one buffer."""
    T, HQ, HK, D = 9, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    h = torch.randn((T, HQ + 2 * HK, D), generator=g).to(F16).to(dev)
    pos, f = torch.arange(T, dtype=torch.int32, device=dev), inv_freq(D).to(dev)
    slots = torch.arange(20, 20 + T, dtype=torch.int32, device=dev)
    want = qm.KvCache.new(3, HK, 16, D, F16)
    q = qm.kv_append(h.view(T, -1), HQ, want, slots, pos, f)
    x = torch.full((T, 1000), 7.0, dtype=F16, device=dev)
    x[:, 8:8 + HK * D] = h[:, HQ + HK:].reshape(T, -1)  # values first
    for i in range(HK):
        x[:, 200 + 80 * i:264 + 80 * i] = h[:, HQ + i]
    for i in range(HQ):
        x[:, 400 + 128 * i:464 + 128 * i] = h[:, i]
    both = torch.zeros((3, HK, 16, 2, D), dtype=F16, device=dev)
    kv = qm.KvCache(both[:, :, :, 0], both[:, :, :, 1])
    got = qm.kv_append(x, HQ, kv, slots, pos, f, q_off=400, q_hs=128, k_off=200, k_hs=80, v_off=8)
    assert torch.equal(got, q) and torch.equal(kv.k, want.k) and torch.equal(kv.v, want.v)
    z, kv = h.clone().view(T, -1), qm.KvCache.new(3, HK, 16, D, F16)
    qm.kv_append(z, HQ, kv, slots, pos, f, q=z[:, :HQ * D])
    assert torch.equal(z[:, :HQ * D].view(T, HQ, D), q) and torch.equal(kv.k, want.k) and torch.equal(z[:, HQ * D:], h.view(T, -1)[:, HQ * D:])


def test_tokens_without_a_place(qm, dev):
    """Slots outside the cache: the token's query is computed, nothing is stored anywhere."""
    T, HQ, HK, D = 6, 2, 1, 64
    x = torch.randn((T, (HQ + 2 * HK) * D), generator=torch.Generator().manual_seed(3)).to(dev)
    pos, f = torch.arange(T, dtype=torch.int32, device=dev), inv_freq(D).to(dev)
    slots = torch.tensor([-1, 5, 32, 2 ** 31 - 1, -2 ** 31, 31], dtype=torch.int32, device=dev)
    for ct in (BF16, E4M3):
        kv = qm.KvCache.new(4, HK, 16, D, ct, mean=True)
        part = qm.KvCache(kv.k[1:3], kv.v[1:3], *([None, None] if ct != E4M3 else [kv.k_scale[1:3], kv.v_scale[1:3]]), kv.mean[1:3])
        q = qm.kv_append(x, HQ, part, slots, pos, f)
        assert q.float().abs().sum(2).min() > 0
        raw = kv.k.view(torch.uint8 if ct == E4M3 else BF16).float()
        used = raw.abs().sum((1, 3)).cpu() > 0
        assert used.nonzero().tolist() == [[1, 5], [2, 15]]
        assert kv.mean[2].any() and not kv.mean[:2].any() and not kv.mean[3].any()


def test_special_values(qm, dev):
    """Heads of zeros and below 2^-100, infinities and NaN in an 8-bit cache; infinities and NaN stay in their head and token."""
    D, HK = 64, 5
    x = torch.randn((1, 2 * HK * D), generator=torch.Generator().manual_seed(4))
    v = x[0, HK * D:].view(HK, D)
    v[0] = 0.0
    v[1] *= 2.0 ** -110
    v[2, 7] = float("inf")
    v[3, 9] = float("nan")
    kv = qm.KvCache.new(1, HK, 16, D, E4M3)
    f, p = inv_freq(0).to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    qm.kv_append(x.to(dev), 0, kv, torch.tensor([3], dtype=torch.int32, device=dev), p, f)
    got, sc = kv.v[0, :, 3].float().cpu(), kv.v_scale[0, :, 3].cpu()
    assert not got[:2].any() and not sc[:2].any()
    assert torch.isinf(sc[2]) and torch.isnan(got[2, 7]) and torch.isnan(got[3, 9]) and torch.isfinite(sc[3])
    keep = torch.arange(D) != 9
    assert torch.isfinite(got[3, keep]).all()
    assert torch.allclose(got[4].double() * sc[4].double(), v[4].double(), rtol=2.0 ** -4, atol=float(v[4].abs().max()) * 2.0 ** -10)


def test_no_tokens(qm, dev):
    kv = qm.KvCache.new(2, 1, 16, 64, BF16)
    f = inv_freq(64).to(dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert qm.kv_append(torch.zeros((0, 256), device=dev), 2, kv, none, none, f).shape == (0, 2, 64)


def test_graph_and_streams(qm, dev):
    """Captured once, replayed for the next tokens: slots and positions are read at the replay."""
    T, HQ, HK, D, page = 4, 4, 2, 128, 16
    x = torch.randn((T, (HQ + 2 * HK) * D), device=dev)
    f = inv_freq(D).to(dev)
    pos, slots = torch.arange(T, dtype=torch.int32, device=dev), torch.arange(T, dtype=torch.int32, device=dev) * page + 13
    kv, eager = qm.KvCache.new(T, HK, page, D, E4M3, mean=True), qm.KvCache.new(T, HK, page, D, E4M3, mean=True)
    q = torch.empty((T, HQ, D), dtype=BF16, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qm.kv_append(x, HQ, kv, slots, pos, f, q=q)
    for step in range(3):  # (the third fills the pages)
        x.normal_()
        graph.replay()
        want = qm.kv_append(x, HQ, eager, slots, pos, f)
        torch.cuda.synchronize()
        assert torch.equal(q, want) and torch.equal(kv.mean, eager.mean) and kv.mean.any() == (step == 2)
        for a, b in ((kv.k, eager.k), (kv.v, eager.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(kv.k_scale, eager.k_scale)
        pos.add_(1)
        slots.add_(1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = qm.KvCache.new(T, HK, page, D, E4M3, mean=True)
    with torch.cuda.stream(s):
        slots.sub_(1)
        qm.kv_append(x, HQ, other, slots, pos.sub_(1), f)
    s.synchronize()
    pg, at = (slots // page).long(), (slots % page).long()
    assert torch.equal(other.k.view(torch.uint8)[pg, :, at], eager.k.view(torch.uint8)[pg, :, at])


def test_caches_past_32_bit_offsets(qm, dev):
    D, page, HK = 128, 64, 1
    pages = (2 ** 32 + 2 ** 28) // (page * D * 2)
    k, v = (torch.zeros((pages, HK, page, D), dtype=BF16, device=dev) for _ in range(2))
    kv = qm.KvCache(k, v)
    x = torch.randn((2, 3 * D), generator=torch.Generator().manual_seed(5)).to(dev)
    f, p = inv_freq(D).to(dev), torch.arange(2, dtype=torch.int32, device=dev)
    slots = torch.tensor([pages * page - 1, 7], dtype=torch.int32, device=dev)
    qm.kv_append(x, 1, kv, slots, p, f)
    small = qm.KvCache.new(2, HK, page, D, BF16)
    qm.kv_append(x, 1, small, torch.tensor([2 * page - 1, 7], dtype=torch.int32, device=dev), p, f)
    assert torch.equal(k[-1], small.k[1]) and torch.equal(k[0], small.k[0]) and torch.equal(v[-1], small.v[1])
    assert int((k != 0).any(3).sum()) == 2
