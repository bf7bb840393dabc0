"""Calls on a stream that they name while torch's current stream is busy and works on memory that it has given back."""
import pytest
import torch

from tests import kv_plain as K
from tests.test_gpu_kv_append import inv_freq

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def keep_busy():
    """Some 20 ms of work on the current stream, then a copy of `t`, whose memory goes back to the allocator at once."""
    m = torch.randn((8192, 8192), device="cuda").to(BF16)
    out = torch.empty_like(m)

    def call(shape, dtype):
        for _ in range(20):
            torch.mm(m, m, out=out)
        t = torch.full(shape, 3, dtype=dtype, device="cuda")
        return t.clone()
    return call


def both(busy, f, shape, dtype):
    """f(stream) on a busy current stream and by itself: the same bits; the current stream's work is as it was."""
    s = torch.cuda.Stream()
    want = f(None)
    torch.cuda.synchronize()
    for _ in range(3):
        copy = busy(shape, dtype)
        got = f(s.cuda_stream)
        s.synchronize()
        now = [t.clone() for t in got]  # (the current stream's turn comes after its work)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(now, want))
        assert bool((copy == 3).all())


def test_attention(qm, dev, keep_busy):
    cache = K.Cache(40, 2, 16, 64, BF16, 1)
    _, ln, table, _ = K.batch([100, 70], [60, 3], 16, 40, 1)
    start = torch.tensor([2, 62, 65], dtype=torch.int32, device=dev)  # (rows of no sequence in front and behind)
    q = torch.randn((70, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    kv, ln, table = cache.on(qm, dev), ln.to(dev), table.to(dev)
    sel = torch.arange(6, dtype=torch.int32, device=dev).expand(70, 2, 6).contiguous()
    both(keep_busy, lambda s: [qm.attn_prefix(q, kv, ln, table, start=start, stream=s)], (70, 4, 64), BF16)
    both(keep_busy, lambda s: [qm.attn_pages(q, kv, ln, table, sel, start=start, out=F32, stream=s)], (70, 4, 64), F32)
    both(keep_busy, lambda s: [qm.attn_prefix(q[:2], kv, ln, table, stream=s)], (2, 4, 64), BF16)


def test_choice(qm, dev, keep_busy):
    cache = K.Cache(130, 2, 16, 64, BF16, 3, mean=True)
    _, ln, table, _ = K.batch([1000, 700], [6, 3], 16, 130, 3)
    start = torch.tensor([2, 8, 11], dtype=torch.int32, device=dev)
    q = torch.randn((14, 4, 64), generator=torch.Generator().manual_seed(4)).to(BF16).to(dev)
    kv, ln, table = cache.on(qm, dev), ln.to(dev), table.to(dev)
    both(keep_busy, lambda s: [qm.select_pages(q, kv, ln, table, 9, start=start, stream=s)], (14, 2, 9), torch.int32)
    # its own workspace is nobody else's before it is done: the next tensor of that size on the current stream
    n = qm.select_workspace(kv, 14, table.size(1)).numel()
    want = qm.select_pages(q, kv, ln, table, 9, start=start)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        got = qm.select_pages(q, kv, ln, table, 9, start=start, stream=s.cuda_stream)
        other = torch.full((n,), 0xFF, dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and bool((other == 0xFF).all())


def test_appending(qm, dev, keep_busy):
    x = torch.randn((5, 8 * 64), generator=torch.Generator().manual_seed(5)).to(BF16).to(dev)
    kv, i, f = qm.KvCache.new(2, 2, 16, 64, BF16), torch.arange(5, dtype=torch.int32, device=dev), inv_freq(64).to(dev)
    both(keep_busy, lambda s: [qm.kv_append(x, 4, kv, i, i, f, stream=s), kv.k, kv.v], (5, 4, 64), BF16)


def test_producers_and_the_rotation(qm, dev, keep_busy):
    x = torch.randn((64, 512), generator=torch.Generator().manual_seed(6)).to(dev)
    pos, f = torch.arange(64, dtype=torch.int32, device=dev), inv_freq(64).to(dev)
    raw = lambda ts: [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in ts]  # noqa: E731
    both(keep_busy, lambda s: raw(qm.quantize_fp8(x, stream=s)), (64, 512), torch.uint8)
    both(keep_busy, lambda s: qm.quantize_act(x, stream=s), (64, 512), torch.int8)
    both(keep_busy, lambda s: qm.qk_norm_rope(x, 4, 4, 64, pos, f, stream=s), (64, 4, 64), F32)
