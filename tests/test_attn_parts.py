"""How many parts of 16 bits a weight is held in for the second product, where a bound for sums of many keys would not tell: two keys, of which one has the weight 1
and the value 0 and the other the value 1, so that the result is w / (1 + w) and little else is rounded.

The bound, relative, in units of 2^-24: log2 e, its product (an 8-bit key's scale's too) and the difference to the maximum 3 |logit|; the exponential 4; the parts' sums
on the matrix pipe, which may lose a whole step each, 6; 1 + w, its reciprocal, the product and the result 4; two to spare. And what the parts leave, half a step to the
power of their number. A part less leaves 2^-16 (bf16) or 2^-11 (f16) of a weight at most, of hundreds of rows nearly that."""
import pytest
import torch

from tests import fp8_plain as P

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
# q, cache, result, parts
KINDS = [(BF16, BF16, F32, 3), (F16, F16, F32, 2), (BF16, E4M3, F32, 3), (F16, E4M3, F32, 3), (F16, E4M3, F16, 2), (BF16, BF16, BF16, 1), (F16, F16, F16, 1)]


def logits(T, HQ, dtype):
    return -(torch.rand((T, HQ), generator=torch.Generator().manual_seed(T)) * 4 + 0.05).to(dtype)


def bound(a, cache, out, parts):
    return (3 * a.double().abs() + 16) * P.U32 + P.HALF[F16 if cache == F16 else BF16] ** parts + (P.HALF[out] if out != F32 else 0)


def close(o, a, cache, out, parts):
    """o [T, HQ, ...] against the sigmoid of the logits."""
    want = torch.sigmoid(a.double()).view(*a.shape, *[1] * (o.dim() - 2))
    return bool(((o.double().cpu() - want).abs() <= want * bound(a, cache, out, parts).view(want.shape)).all())


@pytest.mark.parametrize("q,cache,out,parts", KINDS)
def test_a_part_less_would_be_seen(q, cache, out, parts):
    """The arithmetic in 32 bits, with the parts that there are and with one less."""
    a = logits(40, 8, q)
    w = torch.exp(a.float())
    pipe, left, held = F16 if cache == F16 else BF16, w * (64 if cache == F16 else 1), torch.zeros_like(w)
    for n in range(parts):
        if n == parts - 1:
            assert n == 0 or not close((held / (64 if cache == F16 else 1) / (1 + w)).to(out), a, cache, out, parts)
        held += left.to(pipe).float()
        left = left - left.to(pipe).float()
    assert close((held / (64 if cache == F16 else 1) / (1 + w)).to(out), a, cache, out, parts)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("q,cache,out,parts", KINDS)
def test_parts(qm, dev, q, cache, out, parts, D, T):
    """A few rows and many (by small tiles and by large ones), that see two keys of a prefix."""
    HQ, HK = 8, 2
    kv = qm.KvCache.new(2, HK, 16, D, cache)
    k, v = torch.zeros((2, HK, 16, D)), torch.zeros((2, HK, 16, D))
    k[1, :, 1, 0] = 1
    v[1, :, 1] = 1
    for to, t in ((kv.k, k), (kv.v, v)):
        to.view(torch.uint8 if cache == E4M3 else cache).copy_(t.to(cache).view(torch.uint8) if cache == E4M3 else t)
    for s in (kv.k_scale, kv.v_scale):
        if s is not None:
            s.fill_(1)
    for HQn in (2, HQ):
        a = logits(T, HQn, q)
        x = torch.zeros((T, HQn, D), dtype=q)
        x[..., 0] = a
        i32 = lambda *t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
        o = qm.attn_prefix(x.to(dev), kv, i32(0), i32([0]), start=i32(0, T), prefix=i32(1), prefix_len=2, scale=1.0, out=out)
        assert close(o, a, cache, out, parts)
