"""Calls of the paged-cache operators one after the other: lengths handed on
from eviction to eviction, buffers on other streams, batches without a
sequence."""
import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu


def _cache(seed, B, hk, d, page, top, dtype, dev, lens):
    per = max(1, -(-top // page))
    K, V = R.pool(seed, B * per + 2, hk, page, d, dtype, dev)
    return rkv.PagedCache(K, V, R.table(seed + 1, B, per, B * per + 2, dev), torch.tensor(lens, dtype=torch.int32, device=dev))


def test_evictions_in_a_row_hand_their_lengths_on(cuda):
    """new_lens is copied into the cache's lens before the next call; taken as
    the cache's lens itself it is refused before anything is changed, since
    the call would overwrite what it reads."""
    B, HK, D, n = 2, 2, 64, 300
    c = _cache(1, B, HK, D, 16, n, torch.bfloat16, cuda, [300, 150])
    lens = c.lens
    g = torch.Generator(device=cuda).manual_seed(3)
    W = torch.rand((B, HK, n), generator=g, device=cuda)
    first = rkv.WeightEvictor(HK, n, B, 200, cuda, sinks=2, recent=8)
    second = rkv.WeightEvictor(HK, n, B, 120, cuda, sinks=2, recent=8)
    _, new = first(c, W)
    assert new.tolist() == [200, 150]
    c.lens = new
    before = [t.clone() for t in (c.K, c.V, W, new, first.kept)]
    with pytest.raises(ValueError, match="copy"):
        first(c, W)
    assert all(torch.equal(a, b) for a, b in zip(before, (c.K, c.V, W, new, first.kept)))
    second(c, W)  # another evictor's own lengths are no trouble
    assert second.new_lens.tolist() == [120, 120] and new.tolist() == [200, 150]
    c.lens = lens
    lens.copy_(second.new_lens)
    w0 = W.clone()
    kept, new = rkv.WeightEvictor(HK, n, B, 50, cuda)(c, W)
    assert new.tolist() == [50, 50]
    assert kept[..., :50].tolist() == R.kept_lists(w0, [120, 120], 50, 0, 0)


def _tensors(o):
    return [t for t in vars(o).values() if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("kind", ["decoder", "evictor", "prefill"])
def test_buffers_outlive_their_object_while_a_call_on_another_stream_runs(kind, cuda):
    """An object made here, called on another stream that is still busy, and
    dropped: its workspace and outputs are not handed to new tensors (which are
    only allocated here, never written) until the call has run."""
    B, H, HK, D, n = 2, 4, 2, 64, 200
    c = _cache(5, B, HK, D, 16, n, torch.bfloat16, cuda, [n, 90])
    g = torch.Generator(device=cuda).manual_seed(6)
    W = torch.rand((B, HK, n), generator=g, device=cuda)
    Q, K, V = (torch.randn((B, h, n, D), generator=g, device=cuda).to(torch.bfloat16) for h in (H, HK, HK))
    q, out = Q[:, :, 0].contiguous(), torch.zeros_like(Q)
    s = torch.cuda.Stream()
    for cycles in (1000, 200_000_000):  # first to load and allocate, which waits for the device; then about 100 ms
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(cycles)
        if kind == "decoder":
            o = rkv.PagedDecoder(H, HK, D, n, B, cuda, weights=True)
            o(q, c, W, stream=s.cuda_stream)
        elif kind == "evictor":
            o = rkv.WeightEvictor(HK, n, B, 64, cuda)
            o(c, W, stream=s.cuda_stream)
        else:
            o = rkv.SinkAttention(device=cuda)
            o(Q, K, V, out=out, stream=s.cuda_stream)
        mine = [(t.data_ptr(), t.numel() * t.element_size()) for t in _tensors(o)]
        assert mine
        del o
        new = [torch.empty(size, dtype=torch.uint8, device=cuda) for _, size in mine for _ in range(4)]
        busy = not s.query()
    assert busy, "the call ended too early to show anything"
    for t in new:
        for at, size in mine:
            assert t.data_ptr() + t.numel() <= at or at + size <= t.data_ptr()
    torch.cuda.synchronize()


def test_a_batch_without_a_sequence(cuda):
    """Every call of the paged cache takes an empty batch and does nothing."""
    H, HK, D, n = 4, 2, 64, 50
    K, V = R.pool(8, 6, HK, 16, D, torch.bfloat16, cuda)
    K0 = K.clone()
    c = rkv.PagedCache(K, V, torch.empty((0, 4), dtype=torch.int32, device=cuda), torch.empty(0, dtype=torch.int32, device=cuda))
    k = torch.empty((0, 3, HK, D), dtype=torch.bfloat16, device=cuda)
    rkv.paged_append(c, k, k)
    W = torch.empty((0, HK, n), device=cuda)
    assert rkv.PagedDecoder(H, HK, D, n, 0, cuda, weights=True)(k[:, 0].repeat(1, 2, 1), c, W).shape == (0, H, D)
    kept, new = rkv.WeightEvictor(HK, n, 0, 20, cuda)(c, W)
    assert kept.shape == (0, HK, 20) and new.shape == (0,)
    assert rkv.SinkAttention(device=cuda)(*(torch.empty((0, h, 8, D), dtype=torch.bfloat16, device=cuda) for h in (H, HK, HK))).shape[0] == 0
    torch.cuda.synchronize()
    assert torch.equal(K, K0)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 256)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_decode_keeps_non_finite_values_where_they_are(dtype, D, bad, cuda):
    """In a visible row of V: in its column of its KV head's outputs, nowhere
    else.  In a visible row of K: in its KV head's outputs."""
    B, H, HK, n = 1, 6, 3, 700
    c = _cache(11, B, HK, D, 16, n, dtype, cuda, [n])
    g = torch.Generator(device=cuda).manual_seed(12)
    q = torch.randn((B, H, D), generator=g, device=cuda).to(dtype)
    dec, ref = (rkv.PagedDecoder(H, HK, D, n, B, cuda) for _ in range(2))
    ref(q, c)
    at, row = c.block_table[0, 20].long(), 7
    c.V[at, 1, row, 5] = bad
    dec(q, c)
    hit = torch.zeros_like(dec.O, dtype=torch.bool)
    hit[0, 2:4, 5] = True
    assert not bool(dec.O[hit].isfinite().any()) and torch.equal(dec.O[~hit], ref.O[~hit]) and torch.equal(dec.lse, ref.lse)
    c.V[at, 1, row, 5] = 1.0
    ref(q, c)
    c.K[at, 1, row, 5] = bad
    dec(q, c)
    assert torch.equal(dec.O[0, :2], ref.O[0, :2]) and torch.equal(dec.O[0, 4:], ref.O[0, 4:])
