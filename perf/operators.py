"""Performance cases of the 8-bit floating point products and of the q/k norm + rotation, through arcinfer_amd.qmatmul.

Kinds of case (a dict of plain values):
  gemm  one product of M tokens: e4m3 activations with a scale per 128 values, a weight [N][K] of e4m3 with a scale per
        128 x 128 block, C [M][N] in `out`
  prod  a producer of such activations from rows in `x`: op "rows" (the rows themselves), "rmsnorm", "silu" or "gelu"
        (the gate of a gated FFN times the up half). Outputs: the e4m3 rows and their scales
  rope  the query and key heads of QKV rows [q heads | k heads | v heads]: RMS norm of each head (norm), then the rotation
        of its first `rot` elements by positions of `axes` axes. Outputs: q and k

Weights are N(0, 0.02) rows, activations N(0, 1) rows with 1 % outlier channels, both scaled per block to the e4m3 range.
"""
import math

import torch

own = False

EPS = 1e-6
TOP = 448.0  # the largest e4m3 value
TINY = 2.0 ** -100  # blocks whose largest value is below this are held as zeros
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the smallest product: one attention-sized projection of one decoding token
        {"name": "gemm_decode1_4096", "kind": "gemm", "N": 4096, "K": 4096, "M": 1, "out": "f32"},
        # verification of five drafted tokens: the gate projection of an FFN
        {"name": "gemm_verify5_ffn", "kind": "gemm", "N": 17408, "K": 5120, "M": 5, "out": "f32"},
        # a batch of 48 decoding sequences: the down projection, long rows
        {"name": "gemm_batch48_down", "kind": "gemm", "N": 5120, "K": 17408, "M": 48, "out": "bf16"},
        # a short prompt of ragged length on a projection whose rows end inside a scale block
        {"name": "gemm_prompt333", "kind": "gemm", "N": 5184, "K": 5120, "M": 333, "out": "f32"},
        # a medium prompt: the down projection
        {"name": "gemm_prompt777_down", "kind": "gemm", "N": 5120, "K": 17408, "M": 777, "out": "bf16"},
        # a long prompt: the gate projection
        {"name": "gemm_prompt4096", "kind": "gemm", "N": 17408, "K": 5120, "M": 4096, "out": "bf16"},
        # the norm before a projection, five drafted tokens
        {"name": "rmsnorm_5", "kind": "prod", "op": "rmsnorm", "M": 5, "K": 5120, "x": "f32"},
        # the gated activation between the FFN products of a 2K prompt
        {"name": "swiglu_2048", "kind": "prod", "op": "silu", "M": 2048, "K": 17408, "x": "bf16"},
        # four decoding tokens, heads of 256 of which a quarter turns
        {"name": "rope_decode4", "kind": "rope", "T": 4, "HQ": 24, "HK": 4, "D": 256, "rot": 64, "pairs": "halves",
         "axes": 1, "order": "blocks", "norm": True, "x": "f32", "out": "f32"},
        # a long prompt of packed sequences, whole heads of 128
        {"name": "rope_prompt4096", "kind": "rope", "T": 4096, "HQ": 32, "HK": 8, "D": 128, "rot": 128,
         "pairs": "halves", "axes": 1, "order": "blocks", "norm": True, "x": "bf16", "out": "bf16"},
        # text and an image in one prompt: time, height and width in turns
        {"name": "rope_axes3_777", "kind": "rope", "T": 777, "HQ": 24, "HK": 4, "D": 256, "rot": 64, "pairs": "halves",
         "axes": 3, "order": "turns", "norm": True, "x": "f32", "out": "bf16"},
        # the patches of one large image in a vision encoder: height and width, no norm
        {"name": "rope_axes2_image", "kind": "rope", "T": 4899, "HQ": 16, "HK": 16, "D": 80, "rot": 80,
         "pairs": "halves", "axes": 2, "order": "blocks", "norm": False, "x": "bf16", "out": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(("gemm", "gemm", "gemm", "prod", "rope", "rope"))
    if kind == "gemm":
        # tokens from one to a long prompt; any number of rows; rows of whole blocks, or ending inside one
        M = rng.choice((rng.randint(1, 16), _log_int(rng, 17, 4096), _log_int(rng, 17, 4096)))
        return {"kind": kind, "N": _log_int(rng, 512, 17408, rng.choice((1, 16, 128))),
                "K": _log_int(rng, 1024, 5120 if M > 1024 else 17408, rng.choice((8, 128, 128))), "M": M,
                "out": rng.choice(("f32", "bf16", "bf16", "f16"))}
    if kind == "prod":
        return {"kind": kind, "op": rng.choice(("rows", "rmsnorm", "silu", "gelu")), "M": _log_int(rng, 1, 2048),
                "K": _log_int(rng, 512, 17408, rng.choice((1, 32, 128))), "x": rng.choice(("f32", "bf16", "f16"))}
    D = rng.choice((64, 80, 96, 128, 192, 256))
    axes = rng.choice((1, 1, 2, 3))
    HK = rng.choice((1, 2, 4, 8))
    HQ = HK * rng.choice((1, 3, 4, 8))
    T = _log_int(rng, 1, min(8192, 4096 * 40 * 128 // ((HQ + HK) * D)))
    return {"kind": kind, "T": T, "HQ": HQ, "HK": HK, "D": D,
            "rot": rng.choice((D, D, D // 2, D // 4 * 2)), "pairs": rng.choice(("halves", "halves", "adjacent")),
            "axes": axes, "order": rng.choice(("blocks", "turns")), "norm": rng.random() < 0.75,
            "x": rng.choice(("f32", "bf16", "f16")), "out": rng.choice(("f32", "bf16", "f16"))}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _up(n, to):
    return (n + to - 1) // to * to


def _rows(M, K, seed):
    """f32 rows, 1 % of the channels 20 times larger."""
    g = _gen(seed)
    x = torch.randn((M, K), generator=g, device="cuda")
    ch = torch.randperm(K, generator=g, device="cuda")[:max(1, K // 100)]
    x[:, ch] *= 20.0
    return x


def _weight(N, K, seed):
    """A checkpoint's tensors: e4m3 [N][K] and the f32 scale of each 128 x 128 block, the last ones cut."""
    Np, Kp = _up(N, 128), _up(K, 128)
    w = torch.zeros((Np, Kp), device="cuda")
    w[:N, :K] = torch.randn((N, K), generator=_gen(seed), device="cuda").mul_(0.02)
    b = w.view(Np // 128, 128, Kp // 128, 128)
    sc = b.abs().amax((1, 3)) / TOP
    return b.div_(sc[:, None, :, None]).view(Np, Kp)[:N, :K].to(torch.float8_e4m3fn).contiguous(), sc


def _acts(M, K, seed):
    """Rows as the producers leave them: e4m3 [M_stride][Kp] and scales [Kp / 128][M_stride], zeros in the padding."""
    Ms, Kp = _up(M, 16), _up(K, 128)
    x = torch.zeros((Ms, Kp), device="cuda")
    x[:M, :K] = _rows(M, K, seed)
    b = x.view(Ms, Kp // 128, 128)
    sc = b.abs().amax(2) / TOP
    q = (b / torch.where(sc > 0, sc, 1.0)[:, :, None]).clamp_(-TOP, TOP)
    return q.view(Ms, Kp).to(torch.float8_e4m3fn), sc.t().contiguous()


def _sections(case):
    """Pairs for each axis: the first has what the others leave."""
    n, pairs = case["axes"], case["rot"] // 2
    return [pairs - (n - 1) * (pairs // n)] + [pairs // n] * (n - 1)


def _axis_of(case):
    """The axis of each pair: sections one behind the other, or the axes taking turns as far as their sections reach."""
    n, sec = case["axes"], _sections(case)
    i = torch.arange(case["rot"] // 2, device="cuda")
    if case["order"] == "turns":
        return torch.where(i < n * torch.tensor(sec, device="cuda")[i % n], i % n, 0)
    return torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(sec, device="cuda"))


def _positions(case, seed):
    """int32 [axes][T]: packed sequences of different lengths, the last one a chunk far into a long context; with several
    axes the patches of an image behind a few tokens of text."""
    T, axes = case["T"], case["axes"]
    t = torch.arange(T)
    if axes == 1:
        p = torch.where(t < T // 3, t, t - T // 3)
        p = torch.where(t >= T - T // 4, t + 200_000 + seed % 1000, p)[None]
    else:
        side, text = max(1, math.isqrt(T)), (T // 8 if axes == 3 else 0)
        i = (t - text).clamp(min=0)
        grid = [torch.full_like(t, text), text + i // side, text + i % side][3 - axes:]
        p = torch.stack([torch.where(t < text, t, g) for g in grid])
    return p.to(torch.int32).cuda().contiguous()


def _inv_freq(case):
    i = torch.arange(case["rot"] // 2, dtype=torch.float64)
    return (1e6 ** (-2.0 * i / max(1, case["rot"]))).float().cuda()


def prepare(case, seed):
    s = {"case": case}
    k = case["kind"]
    seed = seed * 16
    if k == "gemm":
        s["w8"], s["wsc"] = _weight(case["N"], case["K"], seed)
        s["a8"], s["asc"] = _acts(case["M"], case["K"], seed + 1)
        if own:  # a program keeps the prepared weight and the workspace
            from arcinfer_amd import qmatmul as qm
            s["w"] = qm.Fp8Weight(s["w8"], s["wsc"])
            s["ws"] = qm.gemm_fp8_workspace(s["w"], case["M"])
    elif k == "prod":
        M, K = case["M"], case["K"]
        s["x"] = _rows(M, K * (2 if case["op"] in ("silu", "gelu") else 1), seed).to(DT[case["x"]])
        s["norm"] = torch.rand(K, generator=_gen(seed + 1), device="cuda") + 0.5
    else:
        g = _gen(seed)
        T, D, H = case["T"], case["D"], case["HQ"] + 2 * case["HK"]
        s["x"] = (torch.randn((T, H * D), generator=g, device="cuda") * 2.0).to(DT[case["x"]])
        s["wq"] = torch.rand(D, generator=g, device="cuda") + 0.5
        s["wk"] = torch.rand(D, generator=g, device="cuda") + 0.5
        s["pos"] = _positions(case, seed)
        s["inv_freq"] = _inv_freq(case)
        s["axis"] = _axis_of(case)
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _own(s):
    from arcinfer_amd import qmatmul as qm
    case = s["case"]
    if case["kind"] == "gemm":
        return qm.gemm_fp8(s["w"], s["a8"], s["asc"], M=case["M"], out=DT[case["out"]], ws=s["ws"])
    if case["kind"] == "prod":
        Ms = _up(case["M"], 16)
        if case["op"] == "rows":
            return qm.quantize_fp8(s["x"], M_stride=Ms)
        if case["op"] == "rmsnorm":
            return qm.rmsnorm_fp8(s["x"], s["norm"], EPS, M_stride=Ms)
        return qm.swiglu_fp8(s["x"], case["K"], gelu=case["op"] == "gelu", M_stride=Ms)
    norm = case["norm"]
    return qm.qk_norm_rope(s["x"], case["HQ"], case["HK"], case["D"], s["pos"], s["inv_freq"],
                           wq=s["wq"] if norm else None, wk=s["wk"] if norm else None, eps=EPS,
                           adjacent=case["pairs"] == "adjacent", sections=_sections(case),
                           turns=case["order"] == "turns", out=DT[case["out"]])


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _plain_gemm(s):
    case = s["case"]
    M, N, K = case["M"], case["N"], case["K"]
    a = s["a8"][:M].float().view(M, -1, 128) * s["asc"][:, :M].t()[:, :, None]
    sc = s["wsc"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (a.view(M, -1)[:, :K] @ (s["w8"].float() * sc).t()).to(DT[case["out"]])


def _plain_prod(s):
    case = s["case"]
    M, K = case["M"], case["K"]
    Ms, Kp = _up(M, 16), _up(K, 128)
    x = s["x"].float()
    if case["op"] == "rmsnorm":
        y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["norm"]
    elif case["op"] == "rows":
        y = x
    else:
        g, u = x[:, :K], x[:, K:]
        if case["op"] == "silu":
            y = g / (1.0 + torch.exp(-g)) * u
        else:
            y = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    p = torch.zeros((Ms, Kp), device="cuda")
    p[:M, :K] = y
    b = p.view(Ms, Kp // 128, 128)
    top = b.abs().amax(2)
    top = torch.where(top >= TINY, top, 0.0)
    inv = torch.where(top > 0, TOP / top, 0.0)
    return (b * inv[:, :, None]).view(Ms, Kp).to(torch.float8_e4m3fn), (top / TOP).t().contiguous()


def _turned(x, w, cos, sin, case):
    """x [T, H, D] in 32 bits: normed by w where there is one, and turned."""
    if case["norm"]:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w
    r = case["rot"]
    t = x[..., :r]
    u, v = (t[..., 0::2], t[..., 1::2]) if case["pairs"] == "adjacent" else (t[..., :r // 2], t[..., r // 2:])
    a, b = u * cos - v * sin, v * cos + u * sin
    t = torch.stack([a, b], -1).flatten(-2) if case["pairs"] == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([t, x[..., r:]], -1).to(DT[case["out"]])


def _plain_rope(s):
    case = s["case"]
    T, D, HQ, HK = case["T"], case["D"], case["HQ"], case["HK"]
    # (32 bits lose far positions: a position of 200,000 turns by 0.01 too much or too little)
    angle = (s["pos"].double()[s["axis"]].t() * s["inv_freq"].double())[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = s["x"][:, :HQ * D].reshape(T, HQ, D).float()
    k = s["x"][:, HQ * D:(HQ + HK) * D].reshape(T, HK, D).float()
    return _turned(q, s["wq"], cos, sin, case), _turned(k, s["wk"], cos, sin, case)


def run(state):
    if own:
        return _own(state)
    return {"gemm": _plain_gemm, "prod": _plain_prod, "rope": _plain_rope}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    k = case["kind"]
    if k == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = _up(K, 128) // 128
        b = N * K + 4 * (_up(N, 128) // 128) * kb + M * K + 4 * M * kb + SIZE[case["out"]] * M * N
        return {"bytes": b, "flops": 2.0 * M * N * K}
    if k == "prod":
        M, K = case["M"], case["K"]
        two = 2 if case["op"] in ("silu", "gelu") else 1
        b = two * M * K * SIZE[case["x"]] + M * K + 4 * M * (_up(K, 128) // 128)
        return {"bytes": b + (4 * K if case["op"] == "rmsnorm" else 0), "flops": 6.0 * M * K}
    T, D, H = case["T"], case["D"], case["HQ"] + case["HK"]
    b = T * H * D * (SIZE[case["x"]] + SIZE[case["out"]]) + 4 * case["axes"] * T + 2 * case["rot"]
    return {"bytes": b + (8 * D if case["norm"] else 0), "flops": (4.0 * D + 3.0 * case["rot"]) * T * H}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------
def _exact_gemm(case, seed):
    M, N, K = case["M"], case["N"], case["K"]
    w8, wsc = _weight(N, K, seed)
    a8, asc = _acts(M, K, seed + 1)
    a8, asc, wsc = a8[:M].double(), asc[:, :M].double(), wsc.double()
    y = torch.zeros((M, N), dtype=torch.float64, device="cuda")
    for b in range(0, K, 128):  # one block of 128 at a time: its sum, then both scales
        e = min(K, b + 128)
        part = a8[:, b:e].contiguous() @ w8[:, b:e].double().t().contiguous()
        part *= asc[b // 128][:, None]
        part *= wsc[:, b // 128].repeat_interleave(128)[:N][None, :]
        y += part
    return y


def _exact_prod(case, seed):
    """The e4m3 rows before their rounding (y over the block's scale) and the scales."""
    M, K, op = case["M"], case["K"], case["op"]
    x = _rows(M, K * (2 if op in ("silu", "gelu") else 1), seed).to(DT[case["x"]]).double()
    if op == "rmsnorm":
        w = (torch.rand(K, generator=_gen(seed + 1), device="cuda") + 0.5).double()
        x = x * w / torch.sqrt(x.pow(2).sum(1, keepdim=True) / K + EPS)
    elif op != "rows":
        g, u = x.split(K, 1)
        z = g if op == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
        x = g * u * torch.sigmoid(z)  # (0.5 (1 + tanh z/2) is the sigmoid of z)
    q = torch.zeros((_up(M, 16), _up(K, 128)), dtype=torch.float64, device="cuda")
    sc = torch.zeros((_up(K, 128) // 128, _up(M, 16)), dtype=torch.float64, device="cuda")
    for b in range(0, K, 128):
        top = x[:, b:b + 128].abs().max(1).values
        sc[b // 128, :M] = top / TOP
        q[:M, b:min(K, b + 128)] = x[:, b:b + 128] * (TOP / top)[:, None]
    return q, sc


def _exact_rope(case, seed):
    g = _gen(seed)
    T, D, HQ, HK, rot = case["T"], case["D"], case["HQ"], case["HK"], case["rot"]
    x = (torch.randn((T, (HQ + 2 * HK) * D), generator=g, device="cuda") * 2.0).to(DT[case["x"]]).double()
    ws = [(torch.rand(D, generator=g, device="cuda") + 0.5).double() for _ in range(2)]
    pos, f = _positions(case, seed).double(), _inv_freq(case).double()
    half, n, sec = rot // 2, case["axes"], _sections(case)
    first = [sum(sec[:a]) for a in range(n + 1)]
    out = []
    for h0, h1, w in ((0, HQ, ws[0]), (HQ, HQ + HK, ws[1])):
        z = x[:, h0 * D:h1 * D].reshape(T, h1 - h0, D).clone()
        if case["norm"]:
            z = z * w / torch.sqrt(z.pow(2).sum(2, keepdim=True) / D + EPS)
        z = torch.complex(z, torch.zeros_like(z))
        for i in range(half):  # each pair as one complex number, times e^(i angle)
            if case["order"] == "turns":
                a = i % n if i < n * sec[i % n] else 0
            else:
                a = max(j for j in range(n) if first[j] <= i)
            lo, hi = (2 * i, 2 * i + 1) if case["pairs"] == "adjacent" else (i, i + half)
            e = torch.polar(torch.ones(T, dtype=torch.float64, device="cuda"), pos[a] * f[i])[:, None]
            c = (z[:, :, lo] + 1j * z[:, :, hi]) * e
            z[:, :, lo], z[:, :, hi] = c.real.to(z.dtype), c.imag.to(z.dtype)
        out.append(z.real.contiguous())
    return tuple(out)


def exact(case, seed):
    return {"gemm": _exact_gemm, "prod": _exact_prod, "rope": _exact_rope}[case["kind"]](case, seed * 16)
