"""Plain 64-bit forms of the e4m3 products, their producers and the q/k norm + rotation, on the CPU."""
import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of f32, relative
HALF = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TOP, TINY = 448.0, 2.0 ** -100


def up(n, to):
    return (n + to - 1) // to * to


def random_e4m3(shape, seed, specials=True):
    """Bytes of finite e4m3 values, all of them equally likely (subnormals and both zeros among them)."""
    g = np.random.default_rng(seed)
    b = g.integers(0, 127, shape, dtype=np.uint8) | (g.integers(0, 2, shape, dtype=np.uint8) << 7)
    return torch.from_numpy(b)


def value(b):
    """e4m3 bytes (uint8 or float8 tensor) -> float64."""
    return (b if b.dtype == torch.float8_e4m3fn else b.view(torch.float8_e4m3fn)).float().double()


def gemm(w8, wsc, a8, asc, M):
    """(C, A, L): the product in 64 bits, the same sum over absolute values, and over the largest product that each eight
    neighbouring k could have."""
    N, K = w8.shape
    Kp = up(K, 128)
    w = torch.zeros((N, Kp), dtype=torch.float64, device=w8.device)
    w[:, :K] = value(w8) * wsc.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    a = (value(a8)[:M].view(M, Kp // 128, 128) * asc.double()[:, :M].T[:, :, None]).reshape(M, Kp)
    top = lambda v: v.abs().view(len(v), Kp // 8, 8).amax(2)  # noqa: E731
    return a @ w.T, a.abs() @ w.abs().T, top(a) @ top(w).T


def gemm_bound(A, L, kb, out=torch.float32):
    """Each block: 128 exact products added on the matrix pipe (an addition may lose a whole step, 2 U32 of the sum of
    absolute values), a product of both scales and an fma; then kb additions. Under a C of 16 bits each eight products lose up to
    2^-13 of the largest each, before the C's own rounding."""
    return (2 * 128 + kb + 4) * U32 * A + (0 if out == torch.float32 else 8 * 2.0 ** -13 * L)


def rounding(out, y):
    """The rounding of y to out (f16 below 2^-14: half a step of 2^-24)."""
    return HALF[out] * y.abs() * 1.01 + (2.0 ** -25 if out == torch.float16 else 0)


def quantize32(y):
    """The quantizer's own f32 arithmetic on f32 rows y [M, K] -> (e4m3 values float64 [M, Kp], scales [Kp / 128, M] f32)."""
    M, K = y.shape
    Kp = up(K, 128)
    p = np.zeros((M, Kp), np.float32)
    p[:, :K] = y
    b = p.reshape(M, Kp // 128, 128)
    top = np.abs(b).max(2)
    live = top >= np.float32(TINY)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inv = np.where(live, np.float32(TOP) / top, np.float32(0)).astype(np.float32)
        sc = np.where(live, top / np.float32(TOP), np.float32(0)).astype(np.float32)
        q = torch.from_numpy((b * inv[:, :, None]).astype(np.float32).reshape(M, Kp))
    return value(q.to(torch.float8_e4m3fn)), torch.from_numpy(np.ascontiguousarray(sc.T))


def near_e4m3(q, v, err):
    """Whether every e4m3 value q is v rounded, v known up to err: half a step, 2^-4 of the value (2^-10 below 2^-6)."""
    return bool(((q - v).abs() <= torch.maximum(2.0 ** -4 * v.abs(), torch.tensor(2.0 ** -10, dtype=torch.float64)) + err).all())


def axis_of(i, sections, turns):
    n = len(sections)
    if turns:
        return i % n if i < n * sections[i % n] else 0
    return int(np.searchsorted(np.cumsum(sections), i, side="right"))


def rotated(x, w, eps, pos, inv_freq, sections, turns, adjacent, scale):
    """x [T, H, D] float64 -> (y, B): the result, and |u| + |v| of each element's pair after the norm (its own value where
    it passes), for the error bound."""
    T, H, D = x.shape
    if w is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + eps) * w
    y, B = x.clone(), x.abs().clone()
    half = len(inv_freq)
    for i in range(half):
        lo, hi = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        a = (pos[axis_of(i, sections, turns)].double() * float(inv_freq[i]))[:, None]
        c, s = torch.cos(a) * scale, torch.sin(a) * scale
        u, v = x[:, :, lo], x[:, :, hi]
        y[:, :, lo], y[:, :, hi] = u * c - v * s, v * c + u * s
        B[:, :, lo] = B[:, :, hi] = (u.abs() + v.abs()) * abs(scale)
    return y, B


def norm_error(n, seq):
    """Relative error of x * w / sqrt(mean(x^2) + eps) in f32, of n values: squares added in chains of seq and a tree, half of
    which the root passes on; mean, eps, root, reciprocal and two products, each a rounding (the root and divisions are
    correctly rounded)."""
    return ((seq + np.log2(max(2, n)) + 3) / 2 + 4) * U32
