"""What the paged cache's operators refuse, what a call of nothing does, and the sizes of their workspaces: through the C ABI, without a
GPU (every check comes before the first device call)."""
import ctypes

import pytest

ARG, SHAPE, TYPE, WORKSPACE = 1, 2, 3, 6
F32, F16, BF16, E4M3 = 0, 1, 30, 256


@pytest.fixture()
def p():
    b = (ctypes.c_uint8 * (1 << 20))()
    yield (ctypes.addressof(b) + 255) // 256 * 256
    del b


def cache(qm, p, type=BF16, D=64, heads=2, page=16, pages=4, ps=None, hs=None, ts=None, k=None, v=None, ks=0, vs=0, mean=None, **_):
    ts = D if ts is None else ts
    hs = page * ts if hs is None else hs
    ps = heads * hs if ps is None else ps
    ks, vs = (p + 0x60000 if type == E4M3 and s == 0 else s or None for s in (ks, vs))
    if vs and vs == ks:
        vs += 0x1000
    return qm.QmKv(type, D, heads, page, pages, ps, hs, ts, p + 0x40000 if k is None else k or None, p + 0x50000 if v is None else v or None,
                   ks, vs, mean)


def seqs(qm, p, T=2, B=2, start=None, len=None, table=None, stride=2, **_):
    return qm.QmSeqs(T, B, start, p + 0x70000 if len is None else len or None, p + 0x71000 if table is None else table or None, stride)


CACHE = {"type", "D", "heads", "page", "pages", "ps", "hs", "ts", "k", "v", "ks", "vs", "mean"}
SEQS = {"T", "B", "start", "len", "table", "stride"}


def attn(qm, p, chosen=False, **a):
    kv, s = cache(qm, p, **a), seqs(qm, p, **a)
    d = dict(q=p, qt=BF16, ldq=256, HQ=4, seqs=ctypes.byref(s), kv=ctypes.byref(kv), list=p + 0x72000, n=0 if not chosen else 2, scale=0.1, o=p + 0x10000,
             ot=BF16, ldo=256, ws=p + 0x80000, wsb=0x10000, st=None)
    assert set(a) <= set(d) | CACHE | SEQS
    d.update({k: v for k, v in a.items() if k in d})
    lib = qm.load_library()
    return (lib.qmatmul_attn_pages if chosen else lib.qmatmul_attn_prefix)(*d.values())


def select(qm, p, **a):
    kv, s = cache(qm, p, **{"mean": p + 0x62000, **a}), seqs(qm, p, **{"stride": 4, **a})
    d = dict(q=p, qt=BF16, ldq=256, HQ=4, seqs=ctypes.byref(s), kv=ctypes.byref(kv), kk=3, first=1, last=1, sel=p + 0x20000, ws=p + 0x80000, wsb=0x10000,
             st=None)
    assert set(a) <= set(d) | CACHE | SEQS
    d.update({k: v for k, v in a.items() if k in d})
    return qm.load_library().qmatmul_select_pages(*d.values())


def append(qm, p, rot=64, axes=1, sections=(0, 0, 0, 0), T=2, **a):
    kv, r = cache(qm, p, **a), qm.QmRope(rot, 0, axes, 0, (ctypes.c_int * 4)(*sections), 1.0)
    d = dict(x=p, xt=F32, ldx=512, T=T, q_off=0, q_hs=64, HQ=4, k_off=256, k_hs=64, v_off=384, v_hs=64, wq=None, wk=None, eps=1e-6, rope=ctypes.byref(r),
             pos=p + 0x30000, pst=2, f=p + 0x31000, slots=p + 0x32000, kv=ctypes.byref(kv), q=p + 0x10000, qt=BF16, ldq=256, st=None)
    assert set(a) <= set(d) | CACHE
    d.update({k: v for k, v in a.items() if k in d})
    return qm.load_library().qmatmul_kv_append(*d.values())


CACHES = [(dict(type=2), TYPE), (dict(type=F32), TYPE), (dict(D=8), SHAPE), (dict(D=72), SHAPE), (dict(D=272), SHAPE), (dict(heads=0), SHAPE),
          (dict(page=24), SHAPE), (dict(page=8), SHAPE), (dict(page=512), SHAPE), (dict(pages=0), SHAPE), (dict(pages=2 ** 27), SHAPE),
          (dict(k=0), ARG), (dict(v=0), ARG), (dict(type=E4M3, ks=None), ARG), (dict(type=E4M3, vs=None), ARG), (dict(ts=56), SHAPE), (dict(hs=512), SHAPE),
          (dict(ps=1024), SHAPE), (dict(ps=-4096), SHAPE), (dict(ts=2 ** 26), SHAPE), (dict(ps=2 ** 45), SHAPE), (dict(ts=68), ARG), (dict(hs=1028), ARG)]


@pytest.mark.parametrize("bad,status", CACHES)
def test_caches(qm, p, bad, status):
    if bad.get("D", 64) != 64:
        bad = {**bad, "ldq": 4096, "ldo": 4096}
    assert attn(qm, p, **bad) == status
    assert attn(qm, p, chosen=True, **bad) == status
    if not set(bad) & {"k", "v", "ks", "vs", "ts", "hs", "ps"}:  # (the choice reads means only)
        assert select(qm, p, **{k: v for k, v in bad.items() if k != "ldo"}) == status
    if "D" not in bad:
        assert append(qm, p, **bad) == status


def test_unaligned_caches(qm, p):
    for k in (dict(k=p + 0x40008), dict(v=p + 0x50002), dict(mean=p + 0x62008), dict(type=E4M3, ks=p + 0x60004), dict(type=E4M3, vs=p + 0x60008)):
        assert attn(qm, p, **k) == ARG and append(qm, p, **k) == ARG, k


@pytest.mark.parametrize("chosen", [False, True])
def test_attention(qm, p, chosen):
    call = lambda **k: attn(qm, p, chosen, **k)  # noqa: E731
    assert call(T=0, B=0) == 0 and call(T=0, B=0, q=None, o=None, len=0, table=0) == 0  # (nothing to do)
    assert call(T=0, B=3, start=p + 0x73000) == 0
    assert call(kv=None) == ARG and call(seqs=None) == ARG
    assert call(q=None) == ARG and call(o=None) == ARG and call(len=0) == ARG and call(table=0) == ARG
    assert call(qt=F32) == TYPE and call(qt=F16) == TYPE and call(ot=F16) == TYPE and call(ot=E4M3) == TYPE
    assert call(type=E4M3, qt=F16, ot=BF16) == TYPE
    for bad in (dict(HQ=3), dict(HQ=0), dict(HQ=-2), dict(HQ=65538), dict(ldq=255), dict(ldo=255), dict(T=-1), dict(B=-1), dict(T=3), dict(stride=0),
                dict(stride=2 ** 27)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(q=p + 1), dict(o=p + 0x10001), dict(ot=F32, o=p + 0x10002), dict(len=p + 0x70002), dict(table=p + 0x71001), dict(start=p + 0x73002, T=3),
                dict(ws=p + 0x80010)):
        assert call(**bad) == ARG, bad
    assert call(T=2 ** 24, B=2 ** 24, HQ=65536, ldq=2 ** 30, ldo=2 ** 30, D=16, ws=None) == SHAPE  # (more than a grid holds)
    # outputs and workspaces over inputs
    for bad in (dict(o=p), dict(o=p + 256), dict(o=p + 0x40100), dict(o=p + 0x50000 - 512), dict(o=p + 0x70000), dict(o=p + 0x71000),
                dict(type=E4M3, o=p + 0x60000, k=p + 0x40000), dict(ws=p), dict(ws=p + 0x10000), dict(ws=p + 0x40000), dict(ws=p + 0x70000)):
        assert call(**bad) == ARG, bad


def test_prefix_and_chosen_lists(qm, p):
    assert attn(qm, p, n=5, list=None) == ARG and attn(qm, p, n=-1) == SHAPE and attn(qm, p, n=2 ** 30 + 1) == SHAPE
    assert attn(qm, p, n=5, list=p + 0x72002) == ARG and attn(qm, p, n=5, list=p + 0x10000) == ARG
    assert attn(qm, p, True, list=None) == ARG and attn(qm, p, True, list=p + 0x72002) == ARG and attn(qm, p, True, list=p + 0x10000) == ARG
    assert attn(qm, p, True, n=0) == SHAPE and attn(qm, p, True, n=2 ** 27) == SHAPE


def test_choice(qm, p):
    call = lambda **k: select(qm, p, **k)  # noqa: E731
    assert call(T=0, B=0) == 0
    assert call(mean=None) == ARG and call(kv=None) == ARG and call(seqs=None) == ARG and call(q=None) == ARG and call(sel=None) == ARG
    assert call(qt=F32) == TYPE
    for bad in (dict(kk=0), dict(first=-1), dict(last=0), dict(first=2, last=2), dict(kk=1), dict(first=2 ** 31 - 1), dict(HQ=3), dict(ldq=200), dict(T=3)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(q=p + 1), dict(sel=p + 0x20002), dict(ws=p + 0x80008), dict(sel=p), dict(sel=p + 0x62000), dict(sel=p + 0x71000), dict(ws=p),
                dict(ws=p + 0x62000), dict(sel=p + 0x80000)):
        assert call(**bad) == ARG, bad
    assert call(ws=None) == WORKSPACE and call(wsb=2 * 2 * 4 * 8 - 1) == WORKSPACE
    assert call(T=2 ** 24, B=2 ** 24, stride=2 ** 16) == SHAPE  # (more than a grid holds)
    assert call(T=2 ** 22, B=2 ** 22, stride=2 ** 16) == WORKSPACE


def test_appending(qm, p):
    call = lambda **k: append(qm, p, **k)  # noqa: E731
    assert call(T=0) == 0 and call(T=0, x=None, q=None, slots=None) == 0
    assert call(x=None) == ARG and call(q=None) == ARG and call(slots=None) == ARG and call(pos=None) == ARG and call(f=None) == ARG and call(rope=None) == ARG
    assert call(xt=2) == TYPE and call(qt=E4M3) == TYPE
    for bad in (dict(T=-1), dict(T=2 ** 24), dict(HQ=-1), dict(HQ=65537), dict(rot=66), dict(rot=63), dict(axes=5), dict(axes=2, sections=(16, 15, 0, 0)),
                dict(q_off=-1), dict(k_off=-1), dict(v_off=-1), dict(q_hs=60), dict(k_hs=60), dict(v_hs=60), dict(v_off=385), dict(ldx=500), dict(ldq=255)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(x=p + 2), dict(q=p + 0x10001), dict(slots=p + 0x32002), dict(pos=p + 0x30001), dict(f=p + 0x31002), dict(wq=p + 0x33002),
                dict(wk=p + 0x33001)):
        assert call(**bad) == ARG, bad
    # the queries over what is read, the cache over everything else
    for bad in (dict(q=p + 0x30000), dict(q=p + 0x32000), dict(q=p + 0x40000), dict(q=p + 1024), dict(k=p), dict(v=p + 0x10000), dict(k=p + 0x32000 - 256),
                dict(k=p + 0x50000 - 256), dict(mean=p + 0x40000), dict(mean=p), dict(type=E4M3, ks=p + 0x50000), dict(type=E4M3, vs=p)):
        assert call(**bad) == ARG, bad


def test_workspaces(qm, p):
    """Sizes that grow with neither lengths nor pages; 0 for what cannot be."""
    lib = qm.load_library()
    ref = lambda **k: ctypes.byref(cache(qm, p, **k))  # noqa: E731
    a = lib.qmatmul_attn_workspace_size
    for bad in ((None, 1, 1, 4, 0), (ref(), 0, 1, 4, 0), (ref(), 1, 0, 4, 0), (ref(), 1, 1, 3, 0), (ref(), 1, 1, 0, 0), (ref(), 1, 1, 4, -1),
                (ref(), 1, 1, 4, 2 ** 30 + 1), (ref(D=24), 1, 1, 4, 0)):
        assert a(*bad) == 0
    for type in (BF16, F16, E4M3):
        for D, T, B, HQ, prefix in ((64, 1, 1, 4, 0), (128, 48, 48, 32, 8192), (256, 36, 12, 24, 0), (128, 2251, 3, 32, 1000), (128, 4096, 1, 32, 0),
                                    (16, 1, 1, 2, 2 ** 30), (256, 512, 512, 128, 60000)):
            n = a(ref(type=type, D=D, pages=4), T, B, HQ, prefix)
            assert 0 <= n < 2 ** 28 and n % 256 == 0
            assert n == a(ref(type=type, D=D, pages=2 ** 20), T, B, HQ, prefix)
    assert lib.qmatmul_select_workspace_size(ref(), 3, 100) == 3 * 2 * 100 * 8 // 256 * 256 + (256 if 4800 % 256 else 0)
    assert lib.qmatmul_select_workspace_size(ref(), 0, 100) == 0 and lib.qmatmul_select_workspace_size(ref(), 1, 0) == 0
