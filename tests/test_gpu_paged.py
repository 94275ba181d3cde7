"""The paged KV cache on the GPU: appended rows, one-token attention and
eviction by accumulated weight, each against its plain form in 64 bits
(tests/pagedref.py), and a generation loop over all three."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _cache(seed, B, hk, d, page, top, dtype, dev, layout="hnd", lens=None, extra=3):
    per = max(1, -(-top // page))
    K, V = R.pool(seed, B * per + extra, hk, page, d, dtype, dev, layout)
    tab = R.table(seed + 1, B, per, B * per + extra, dev)
    lens = torch.tensor([top] * B if lens is None else lens, dtype=torch.int32, device=dev)
    return rkv.PagedCache(K, V, tab, lens)


def _query(seed, B, H, d, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn((B, H, d), generator=g, device=dev).to(dtype)


def _check_decode(dec, Q, c, sinks=0, window=0, skip=(), W0=None, W=None):
    O, lse, w, tO, tL, tW = R.decode(Q, c.K, c.V, c.block_table, c.lens, sinks, window, skip)
    assert bool(((dec.O - O).abs() <= tO).all()), float(((dec.O - O).abs() / tO).max())
    inf = lse == -math.inf
    assert torch.equal(inf, dec.lse == -math.inf)
    assert bool(((dec.lse - lse).abs()[~inf] <= tL[~inf]).all())
    if W is not None:
        for b, (x, t) in enumerate(zip(w, tW)):
            n = x.shape[1]
            want = W0[b, :, :n].double() + x
            assert bool(((W[b, :, :n] - want).abs() <= t + 2 * R.EPS * want.abs()).all()), b
            assert torch.equal(W[b, :, n:], W0[b, :, n:])


# (type, D, H, HK, page, lens, sinks, window, layout)
DECODE = [
    ("bf16", 128, 24, 8, 16, [2048], 0, 0, "hnd"),
    ("bf16", 128, 24, 8, 16, [0, 1, 15, 16, 17, 31, 32, 33, 129, 1000], 0, 0, "nhd"),
    ("f16", 128, 24, 8, 32, [3717, 1, 700], 0, 0, "mixed"),
    ("f32", 128, 24, 8, 16, [513, 0, 128], 0, 0, "hnd"),
    ("f32", 64, 8, 8, 24, [4099, 77, 1029], 4, 1024, "nhd"),
    ("bf16", 64, 8, 1, 8, [300, 299, 63], 0, 0, "hnd"),
    ("f16", 64, 16, 2, 1, [67, 5], 3, 7, "hnd"),
    ("bf16", 96, 12, 4, 48, [777, 96, 97], 0, 100, "hnd"),
    ("f16", 80, 5, 5, 16, [257, 40], 33, 1, "mixed"),
    ("bf16", 256, 16, 2, 16, [515, 2], 0, 0, "hnd"),
    ("f32", 256, 24, 2, 64, [130, 64], 4, 64, "nhd"),
    ("f16", 8, 2, 1, 16, [100], 0, 0, "hnd"),
    ("f32", 24, 3, 3, 5, [31, 4], 0, 0, "hnd"),
    ("bf16", 128, 64, 4, 128, [1111, 128], 10, 200, "hnd"),    # 16 query heads a KV head
    ("f16", 128, 40, 2, 16, [400, 19], 0, 0, "hnd"),           # 20
    ("bf16", 248, 6, 3, 16, [333, 0], 0, 0, "hnd"),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, (c[0], "d%d" % c[1], "h%d" % c[2], "k%d" % c[3], "p%d" % c[4], max(c[5])))))
@pytest.mark.parametrize("weights", [False, True])
def test_decode_against_64_bits(case, weights, cuda):
    kind, D, H, HK, page, lens, sinks, window, layout = case
    dt, B, top = TYPES[kind], len(case[5]), max(case[5])
    c = _cache(10, B, HK, D, page, top, dt, cuda, layout, lens)
    Q = _query(12, B, H, D, dt, cuda)
    dec = rkv.PagedDecoder(H, HK, D, top, B, cuda, sinks=sinks, window=window, weights=weights)
    dec.O.fill_(7.0)
    W = W0 = None
    if weights:
        g = torch.Generator(device=cuda).manual_seed(13)
        W0 = torch.rand((B, HK, top + 5), generator=g, device=cuda)
        W = W0.clone()
    dec(Q, c, W)
    torch.cuda.synchronize()
    _check_decode(dec, Q, c, sinks, window, W0=W0, W=W)


def test_decode_large_scores_and_salient_keys(cuda):
    """Rows whose largest score moves late, far apart scores, and one token
    that takes all the weight."""
    B, H, HK, D, n = 2, 24, 8, 128, 1500
    c = _cache(20, B, HK, D, 16, n, torch.bfloat16, cuda)
    c.K.mul_(torch.linspace(0.1, 8.0, c.K.shape[0], device=cuda).to(torch.bfloat16)[:, None, None, None])
    Q = _query(21, B, H, D, torch.bfloat16, cuda) * 4
    W = torch.zeros((B, HK, n), device=cuda)
    dec = rkv.PagedDecoder(H, HK, D, n, B, cuda, weights=True)
    dec(Q, c, W)
    _check_decode(dec, Q, c, W0=torch.zeros_like(W), W=W)
    assert abs(float(W.sum()) - B * H) < 1e-3


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_decode_reads_nothing_that_is_masked(kind, cuda):
    """NaN in rows behind a sequence's end and outside its window, in pages no
    sequence owns, and page numbers behind the end that lie outside the pool."""
    dt, B, H, HK, D, page = TYPES[kind], 3, 24, 8, 128, 16
    lens = [200, 37, 0]
    c = _cache(30, B, HK, D, page, 256, dt, cuda, lens=lens)
    K, V = c.K, c.V
    sinks, window = 4, 50
    want = rkv.PagedDecoder(H, HK, D, 256, B, cuda, sinks=sinks, window=window)
    Q = _query(31, B, H, D, dt, cuda)
    want(Q, c)
    keep = torch.zeros(K.shape[:1] + K.shape[2:3], dtype=torch.bool, device=cuda)
    for b, n in enumerate(lens):
        t = R.seen(n, sinks, window).to(cuda)
        keep[c.block_table[b].long()[t // page], t % page] = True
    bad = ~keep[:, None, :, None]
    K.masked_fill_(bad, math.nan)
    V.masked_fill_(bad, math.inf)
    for b, n in enumerate(lens):
        first = -(-n // page)
        c.block_table[b, first:] = torch.tensor([(-1) ** i * (10 ** 6 + i) for i in range(c.block_table.shape[1] - first)],
                                                dtype=torch.int32, device=cuda)
    got = rkv.PagedDecoder(H, HK, D, 256, B, cuda, sinks=sinks, window=window)
    got(Q, c)
    assert torch.equal(got.O, want.O) and torch.equal(got.lse, want.lse)
    _check_decode(got, Q, c, sinks, window)


def test_decode_leaves_out_pages_outside_the_pool(cuda):
    B, H, HK, D, page, n = 2, 6, 2, 64, 16, 150
    c = _cache(40, B, HK, D, page, n, torch.float16, cuda)
    c.block_table[0, 3] = -1
    c.block_table[1, 0] = c.K.shape[0]
    c.block_table[1, 9] = 2 ** 31 - 1
    skip = {(0, t) for t in range(48, 64)} | {(1, t) for t in range(16)} | {(1, t) for t in range(144, 150)}
    Q = _query(41, B, H, D, torch.float16, cuda)
    W0 = torch.rand((B, HK, n), device=cuda)
    W = W0.clone()
    dec = rkv.PagedDecoder(H, HK, D, n, B, cuda, weights=True)
    dec(Q, c, W)
    _check_decode(dec, Q, c, skip=skip, W0=W0, W=W)
    c.block_table.fill_(-1)  # nothing left
    dec(Q, c)
    assert bool((dec.O == 0).all()) and bool((dec.lse == -math.inf).all())


def test_decode_non_finite_keys_stay_in_their_heads(cuda):
    """An infinite or NaN key that is visible spoils its KV head's outputs
    only, as in the formula."""
    B, H, HK, D, n = 1, 8, 4, 64, 90
    c = _cache(45, B, HK, D, 16, n, torch.bfloat16, cuda)
    Q = _query(46, B, H, D, torch.bfloat16, cuda)
    ref = rkv.PagedDecoder(H, HK, D, n, B, cuda)
    ref(Q, c)
    for h, bad in ((1, math.nan), (2, math.inf)):
        c.K[c.block_table[0, 2].long(), h, 5] = bad
    dec = rkv.PagedDecoder(H, HK, D, n, B, cuda)
    dec(Q, c)
    assert bool(dec.O[0, 2:6].isnan().all())
    assert torch.equal(dec.O[0, :2], ref.O[0, :2]) and torch.equal(dec.O[0, 6:], ref.O[0, 6:])


def test_decode_lengths_are_clamped(cuda):
    """lens beyond max_len or the table, or negative."""
    B, H, HK, D, page = 3, 4, 2, 64, 16
    c = _cache(50, B, HK, D, page, 64, torch.float32, cuda, lens=[1000, 60, -5])
    Q = _query(51, B, H, D, torch.float32, cuda)
    dec = rkv.PagedDecoder(H, HK, D, 50, B, cuda)
    dec(Q, c)
    c.lens = torch.tensor([50, 50, 0], dtype=torch.int32, device=cuda)
    _check_decode(dec, Q, c)
    c.lens = torch.tensor([1000, 64, 3], dtype=torch.int32, device=cuda)
    big = rkv.PagedDecoder(H, HK, D, 5000, B, cuda)
    big(Q, c)
    c.lens = torch.tensor([64, 64, 3], dtype=torch.int32, device=cuda)
    _check_decode(big, Q, c)


def test_decode_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes whose last pages are used."""
    H, HK, D, page = 8, 8, 128, 128
    pages = (1 << 32) // (HK * page * D * 2) + 40
    K = torch.empty((pages, HK, page, D), dtype=torch.bfloat16, device=cuda)
    assert K.numel() * 2 > 1 << 32
    tab = torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, pages - 30, 1]], dtype=torch.int32, device=cuda)
    for p in tab.view(-1).tolist():
        K[p] = torch.randn((HK, page, D), device=cuda).to(torch.bfloat16)
    c = rkv.PagedCache(K, K, tab, torch.tensor([384, 300], dtype=torch.int32, device=cuda))
    Q = _query(55, 2, H, D, torch.bfloat16, cuda)
    dec = rkv.PagedDecoder(H, HK, D, 384, 2, cuda)
    dec(Q, c)
    _check_decode(dec, Q, c)
    # and appended to: the newest row of each sequence
    k = torch.randn((2, HK, D), device=cuda).to(torch.bfloat16)
    rkv.paged_append(c, k, k)
    assert torch.equal(K[pages - 3, :, 127], k[0]) and torch.equal(K[1, :, 43], k[1])


def test_decode_repeats_bit_for_bit_and_in_a_graph(cuda):
    """The same call twice, the call in a captured graph replayed over other
    lengths and queries, and two calls on two streams."""
    B, H, HK, D, page, top = 4, 24, 8, 128, 16, 3000
    c = _cache(60, B, HK, D, page, top, torch.bfloat16, cuda, lens=[3000, 17, 1500, 0])
    Q = _query(61, B, H, D, torch.bfloat16, cuda)
    dec = rkv.PagedDecoder(H, HK, D, top, B, cuda, weights=True)
    W = torch.zeros((B, HK, top), device=cuda)
    dec(Q, c, W)
    first, W1 = dec.O.clone(), W.clone()
    W.zero_()
    dec.O.zero_()
    dec(Q, c, W)
    assert torch.equal(dec.O, first) and torch.equal(W, W1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec(Q, c, W)
    W0 = torch.zeros_like(W)
    for lens, seed in (([3000, 17, 1500, 0], 61), ([1, 2999, 640, 128], 62)):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        Q.copy_(_query(seed, B, H, D, torch.bfloat16, cuda))
        W.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check_decode(dec, Q, c, W0=W0, W=W)
    other = rkv.PagedDecoder(H, HK, D, top, B, cuda)
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = dec.O.clone()
    torch.cuda.synchronize()
    for s, d in zip(streams, (dec, other)):
        for _ in range(3):
            d(Q, c, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(dec.O, want) and torch.equal(other.O, want)


# ---- append --------------------------------------------------------------------
@pytest.mark.parametrize("kind,D,HK,page,layout", [("bf16", 128, 8, 16, "hnd"), ("f16", 64, 2, 24, "nhd"), ("f32", 8, 3, 1, "mixed"),
                                                   ("bf16", 72, 5, 7, "hnd")])
@pytest.mark.parametrize("odd", [False, True])
def test_append_puts_every_row_in_its_place(kind, D, HK, page, layout, odd, cuda):
    """Ragged counts, rows read from a fused buffer (odd: one that starts at an
    odd element), everything else untouched."""
    dt, B, T, top = TYPES[kind], 5, 37, 100
    lens, n_new = [100, 40, 1, 0, 64], [37, 0, 1, 0, 20]
    c = _cache(70, B, HK, D, page, top, dt, cuda, layout, lens)
    K0, V0 = c.K.clone(), c.V.clone()
    flat = torch.randn(B * T * 2 * HK * D + 1, device=cuda).to(dt)
    fused = flat[int(odd): int(odd) + B * T * 2 * HK * D].view(B, T, 2 * HK, D)
    k, v = fused[:, :, :HK], fused[:, :, HK:]
    rkv.paged_append(c, k, v, torch.tensor(n_new, dtype=torch.int32, device=cuda))
    for b in range(B):
        for i in range(n_new[b]):
            t = lens[b] - n_new[b] + i
            p, r = int(c.block_table[b, t // page]), t % page
            K0[p, :, r], V0[p, :, r] = k[b, i], v[b, i]
    assert torch.equal(c.K, K0) and torch.equal(c.V, V0)


def test_append_skips_what_has_no_place(cuda):
    """More rows than the sequence counts, tokens behind the table, page
    numbers outside the pool, counts outside [0, n_rows]."""
    B, HK, D, page = 4, 2, 64, 16
    c = _cache(75, B, HK, D, page, 32, torch.float32, cuda, lens=[2, 40, 32, 20])
    c.block_table[2, 1] = -7
    K0 = c.K.clone()
    k = torch.randn((B, 6, HK, D), device=cuda)
    rkv.paged_append(c, k, k, torch.tensor([6, 6, 6, -3], dtype=torch.int32, device=cuda))
    tab = c.block_table.tolist()
    K0[tab[0][0], :, 0], K0[tab[0][0], :, 1] = k[0, 4], k[0, 5]  # rows 0 .. 3 would be tokens -4 .. -1
    # sequence 1: tokens 34 .. 39 lie behind its two pages; sequence 2: page -7; sequence 3: no rows
    assert torch.equal(c.K, K0)
    rkv.paged_append(c, k[:, :1], k[:, :1], torch.tensor([9, 9, 0, 0], dtype=torch.int32, device=cuda))  # clamped to one row
    K0[tab[0][0], :, 1] = k[0, 0]
    assert torch.equal(c.K, K0)


# ---- eviction ------------------------------------------------------------------------
def _weights(seed, B, HK, top, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn((B, HK, top), generator=g, device=dev).exp()
    return torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.5, (w * 4).round() / 4, w)  # many ties


def _expect_evict(c, K0, V0, W0, lens, kept, out, Ko, Vo, max_len):
    """Pools and weights after the eviction."""
    W = W0.clone()
    for b, per in enumerate(kept):
        for h, k in enumerate(per):
            m = len(k)
            kt = torch.tensor(k, dtype=torch.int64, device=K0.device)
            W[b, h, :m] = W0[b, h, kt]
            W[b, h, m:max_len] = 0
            if m:
                ps, po = c.K.shape[2], out.K.shape[2]
                src, dst = c.block_table[b].long(), out.block_table[b].long()
                i = torch.arange(m, device=K0.device)
                Ko[dst[i // po], h, i % po] = K0[src[kt // ps], h, kt % ps]
                Vo[dst[i // po], h, i % po] = V0[src[kt // ps], h, kt % ps]
    return Ko, Vo, W


EVICT = [
    # type, D, HK, page, lens, budget, sinks, recent, layout, page out
    ("bf16", 128, 8, 16, [2112], 2048, 4, 32, "hnd", 16),
    ("bf16", 128, 8, 16, [3717, 100, 1024, 1025, 0, 1], 1024, 4, 32, "nhd", 64),
    ("f16", 64, 2, 24, [500, 499, 17], 100, 0, 1, "mixed", 7),
    ("f32", 128, 3, 16, [700, 300], 64, 10, 54, "hnd", 16),      # sinks + recent fill the budget
    ("f32", 256, 2, 5, [130, 90], 0, 0, 0, "hnd", 8),            # nothing stays
    ("bf16", 8, 1, 1, [70, 1], 1, 0, 1, "hnd", 1),
    ("f16", 72, 5, 32, [9000, 4097], 4096, 0, 0, "hnd", 32),
    ("bf16", 64, 2, 64, [70001, 20000], 5001, 4, 100, "hnd", 64),
    ("f32", 8, 1, 16, [300000], 100000, 4, 100, "hnd", 128),
    ("f32", 8, 1, 16, [500000, 90000], 100000, 4, 100, "nhd", 128),  # more weights than a cluster's shared memory holds
    ("bf16", 8, 1, 64, [420000], 0, 0, 0, "hnd", 16),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, (c[0], c[1], c[2], max(c[4]), c[5]))))
@pytest.mark.parametrize("inplace", [False, True])
def test_evict_against_the_formula(case, inplace, cuda):
    kind, D, HK, page, lens, budget, sinks, recent, layout, po = case
    dt, B, top = TYPES[kind], len(case[4]), max(case[4])
    c = _cache(80, B, HK, D, page, top, dt, cuda, layout, lens)
    W = _weights(82, B, HK, top + 3, cuda)
    for b, n in enumerate(lens):
        W[b, :, n:] = 1e30  # behind the end: must not be ranked
    K0, V0, W0 = c.K.clone(), c.V.clone(), W.clone()
    want = R.kept_lists(W0, lens, budget, sinks, recent)
    ev = rkv.WeightEvictor(HK, top, B, budget, cuda, sinks=sinks, recent=recent)
    if inplace:
        kept, new = ev(c, W)
        out, Wo = c, W
        Ko, Vo, We = _expect_evict(c, K0, V0, W0, lens, want, c, K0.clone(), V0.clone(), top)
    else:
        out = _cache(84, B, HK, D, po, max(1, min(budget, top)), dt, cuda, "hnd", [0] * B)
        Ko, Vo = out.K.clone(), out.V.clone()
        Wo = torch.full_like(W, -3.0)
        kept, new = ev(c, W, out=out, weights_out=Wo)
        Ko, Vo, We = _expect_evict(c, K0, V0, W0, lens, want, out, Ko, Vo, top)
        We[:, :, top:] = -3.0
        assert torch.equal(c.K, K0) and torch.equal(c.V, V0) and torch.equal(W, W0)
    assert new.tolist() == [min(n, budget) for n in lens]
    for b in range(B):
        for h in range(HK):
            row = kept[b, h].tolist()
            assert row == want[b][h] + [-1] * (len(row) - len(want[b][h])), (b, h)
    assert torch.equal(Wo, We)
    assert torch.equal(out.K, Ko) and torch.equal(out.V, Vo)


def test_evict_ranks_odd_weights(cuda):
    """NaN below everything, -0 as 0, infinities and negative weights in
    order, all weights equal."""
    n, budget = 40, 12
    c = _cache(90, 3, 1, 64, 16, n, torch.bfloat16, cuda)
    W = torch.zeros((3, 1, n), device=cuda)
    W[0, 0, 5:30:3] = math.nan
    W[0, 0, 6] = math.inf
    W[0, 0, 7] = -math.inf
    W[0, 0, 31:36] = -1.0
    W[0, 0, 20:24] = -0.0
    W[0, 0, 36:] = torch.tensor([1e-45, 3e38, -1e-45, 2.0])
    W[1, 0] = 0.25
    W[2, 0] = math.nan
    want = R.kept_lists(W, [n] * 3, budget, 1, 1)
    kept, _ = rkv.WeightEvictor(1, n, 3, budget, cuda, sinks=1, recent=1)(c, W)
    assert kept[:, 0].tolist() == [w[0] for w in want]
    assert want[1][0] == list(range(11)) + [39]


def test_evict_skips_pages_outside_the_pool(cuda):
    n, budget, page = 96, 40, 16
    c = _cache(92, 1, 2, 64, page, n, torch.float32, cuda)
    tab = c.block_table.clone()
    out = _cache(93, 1, 2, 64, page, budget, torch.float32, cuda, lens=[0])
    Ko = out.K.clone()
    W = _weights(94, 1, 2, n, cuda)
    c.block_table[0, 1] = -1
    out.block_table[0, 2] = out.K.shape[0] + 5
    kept, _ = rkv.WeightEvictor(2, n, 1, budget, cuda)(c, W, out=out, weights_out=torch.empty_like(W))
    for h in range(2):
        for i, t in enumerate(kept[0, h].tolist()):
            if t // page != 1 and i // page != 2:
                Ko[int(out.block_table[0, i // page]), h, i % page] = c.K[int(tab[0, t // page]), h, t % page]
    assert torch.equal(out.K, Ko)


def test_evict_into_other_pages_of_the_same_pools(cuda):
    """The destination is a second table over the same pools, as an allocator
    hands out pages; and a captured eviction replayed."""
    B, HK, D, page, n, budget = 2, 4, 64, 16, 320, 96
    K, V = R.pool(95, B * 26, HK, page, D, torch.float16, cuda)
    perm = R.table(96, 1, B * 26, B * 26, cuda)[0]
    src = perm[: B * 20].view(B, 20).contiguous()
    dst = perm[B * 20: B * 26].view(B, 6).contiguous()
    lens = torch.tensor([n, 200], dtype=torch.int32, device=cuda)
    c, out = rkv.PagedCache(K, V, src, lens), rkv.PagedCache(K, V, dst, None)
    W = _weights(97, B, HK, n, cuda)
    Wo = torch.zeros_like(W)
    ev = rkv.WeightEvictor(HK, n, B, budget, cuda, sinks=2, recent=8)
    ev(c, W, out=out, weights_out=Wo)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ev(c, W, out=out, weights_out=Wo)
    W.copy_(_weights(98, B, HK, n, cuda))
    lens.copy_(torch.tensor([150, 310], dtype=torch.int32))
    K0, V0, W0 = K.clone(), V.clone(), W.clone()
    g.replay()
    torch.cuda.synchronize()
    Ko, Vo, We = _expect_evict(c, K0, V0, W0, [150, 310], R.kept_lists(W0, [150, 310], budget, 2, 8), out, K0.clone(), V0.clone(), n)
    assert torch.equal(K, Ko) and torch.equal(V, Vo) and torch.equal(Wo, We)


def test_fresh_objects_on_another_stream(cuda):
    """A decoder and an evictor made and called on another stream while the
    current one is busy: nothing of their making comes behind the calls."""
    B, H, HK, D, page, n, budget = 2, 4, 2, 64, 16, 200, 64
    c = _cache(101, B, HK, D, page, n, torch.bfloat16, cuda, lens=[n, 90])
    out = _cache(102, B, HK, D, page, budget, torch.bfloat16, cuda, lens=[0, 0])
    Q, W = _query(103, B, H, D, torch.bfloat16, cuda), _weights(104, B, HK, n, cuda)
    want = rkv.PagedDecoder(H, HK, D, n, B, cuda)(Q, c)
    kept0, new0 = rkv.WeightEvictor(HK, n, B, budget, cuda, sinks=2)(c, W, out=out, weights_out=torch.zeros_like(W))
    Wo, s = torch.zeros_like(W), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)  # about 25 ms
    dec, ev = rkv.PagedDecoder(H, HK, D, n, B, cuda), rkv.WeightEvictor(HK, n, B, budget, cuda, sinks=2)
    dec(Q, c, stream=s.cuda_stream)
    ev(c, W, out=out, weights_out=Wo, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(dec.O, want) and torch.equal(ev.kept, kept0) and torch.equal(ev.new_lens, new0)


def test_generation_with_evictions(cuda):
    """Prompt rows appended, then 24 steps of append, decode with weights, and
    an eviction in place whenever the cache has grown 8 tokens over its budget;
    every step against the same steps on plain tensors in 64 bits."""
    B, H, HK, D, page, budget, sinks, recent = 3, 12, 4, 64, 16, 48, 2, 6
    prompt, cap = [50, 20, 37], 64
    dt = torch.bfloat16
    c = _cache(100, B, HK, D, page, cap, dt, cuda, lens=prompt)
    g = torch.Generator(device=cuda).manual_seed(101)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda).to(dt)  # noqa: E731
    k, v = rnd(B, 50, HK, D), rnd(B, 50, HK, D)
    rkv.paged_append(c, k, v, torch.tensor(prompt, dtype=torch.int32, device=cuda))
    plain = [[(k[b, :n, h].clone(), v[b, :n, h].clone()) for h in range(HK)] for b, n in enumerate(prompt)]
    W = torch.zeros((B, HK, cap), device=cuda)
    dec = rkv.PagedDecoder(H, HK, D, cap, B, cuda, weights=True)
    ev = rkv.WeightEvictor(HK, cap, B, budget, cuda, sinks=sinks, recent=recent)
    G, evicted = H // HK, 0
    for step in range(24):
        c.lens += 1
        k1, v1, Q = rnd(B, HK, D), rnd(B, HK, D), rnd(B, H, D)
        rkv.paged_append(c, k1, v1)
        W0 = W.clone()
        dec(Q, c, W)
        _check_decode(dec, Q, c, W0=W0, W=W)
        for b in range(B):
            for h in range(HK):
                kk, vv = (torch.cat((x, y[b, h][None])) for x, y in zip(plain[b][h], (k1, v1)))
                plain[b][h] = (kk, vv)
                p = torch.softmax(Q[b, h * G:(h + 1) * G].double() @ kk.double().T / math.sqrt(D), 1)
                assert float((dec.O[b, h * G:(h + 1) * G] - p @ vv.double()).abs().max()) < 1e-4
        if int(c.lens.max()) >= budget + 8:
            lens, before = c.lens.tolist(), W.clone()
            kept, new = ev(c, W)
            c.lens.copy_(new)
            want = R.kept_lists(before, lens, budget, sinks, recent)
            for b in range(B):
                for h in range(HK):
                    assert kept[b, h, : len(want[b][h])].tolist() == want[b][h]
                    t = torch.tensor(want[b][h], device=cuda)
                    plain[b][h] = tuple(x[t] for x in plain[b][h])
            evicted += 1
    assert evicted >= 2
