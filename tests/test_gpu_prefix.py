"""Decode of sequences that share leading tokens, on the GPU, against every
sequence's attention over all of its tokens in 64 bits."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _setup(seed, hk, d, page, groups, dtype, dev, layout="hnd", alone=(), scale=1.0):
    """A cache whose groups share pages.  groups: a list of (shared tokens,
    [every sequence's length]); a sequence shorter than the shared tokens has
    pages of its own.  alone: lengths of sequences of no group, behind them.
    Shared tokens that do not fill a page are copied to every sequence's own."""
    seqs, starts, shared = [], [0], []
    for g, (p, lens) in enumerate(groups):
        seqs += [(g, p, n) for n in lens]
        starts.append(len(seqs))
        shared.append(p)
    seqs += [(-1, 0, n) for n in alone]
    need = lambda n: -(-n // page)  # noqa: E731
    total = sum(p // page for p in shared) + sum(need(n) if n < p else need(n) - p // page for _, p, n in seqs) + 3
    K, V = R.pool(seed, total, hk, page, d, dtype, dev, layout, scale)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    take = lambda n: [order.pop() for _ in range(n)]  # noqa: E731
    whole = [take(p // page) for p in shared]
    per = max(1, max((need(n) for _, _, n in seqs), default=1), max((need(p) for p in shared), default=1))
    table, firsts = [], {}
    for g, p, n in seqs:
        mine = take(need(n)) if n < p else whole[g] + take(need(n) - p // page) if g >= 0 else take(need(n))
        if g >= 0 and n >= p and p % page:  # the rest of the shared tokens, in a page of its own
            at, r = mine[p // page], p % page
            if g in firsts:
                K[at, :, :r], V[at, :, :r] = K[firsts[g], :, :r], V[firsts[g], :, :r]
            else:
                firsts[g] = at
        table.append(mine + [0] * (per - len(mine)))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache = rkv.PagedCache(K, V, i32(table).view(len(seqs), per), i32([n for _, _, n in seqs]))
    return cache, i32(starts), i32(shared)


def _query(seed, B, H, d, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn((B, H, d), generator=g, device=dev).to(dtype)


def _exact(Q, cache, most, skip=()):
    """O, lse (of at most `most` tokens) and bounds on the errors: an exponential's (a dot product of D
    terms, the rounding of its argument), carried through the softmax, and the
    sums' in fp32; with 16 bits a weight's rounding and the output's, and in fp16
    a weight's fixed step of 2^-32 of the row's largest."""
    B, H, D = Q.shape
    HK = cache.K.shape[1]
    G = H // HK
    uT = R.unit(Q.dtype) if Q.dtype != torch.float32 else 0.0
    O = torch.zeros((B, H, D), dtype=torch.float64, device=Q.device)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=Q.device)
    tolO, tolL = torch.zeros_like(O), torch.zeros_like(lse)
    for b in range(B):
        t = torch.tensor([x for x in range(min(most, int(cache.lens[b]))) if (b, x) not in skip], dtype=torch.int64)
        if not len(t):
            continue
        k, v = (R.rows(P, cache.block_table, b, t).double().transpose(0, 1) for P in (cache.K, cache.V))
        q = Q[b].double().view(HK, G, D)
        s = q @ k.transpose(1, 2) / math.sqrt(D)
        mag = q.abs() @ k.abs().transpose(1, 2) / math.sqrt(D)
        m = s.amax(-1, keepdim=True)
        e = torch.exp(s - m)
        total = e.sum(-1, keepdim=True)
        p = e / total
        O[b] = (p @ v).view(H, D)
        lse[b] = (m + total.log()).view(H)
        es = R.EPS * (R.LAM * math.sqrt(D + 2) * mag + 4 * s.abs() + 4 * m.abs() + 8)
        sums = R.EPS * (R.LAM * math.sqrt(len(t)) + 8)
        rel = (p * es).sum(-1, keepdim=True) + sums
        pv = p @ v.abs()
        tol = (p * (es + uT)) @ v.abs() + (rel + sums) * pv + uT * ((p @ v).abs() + 2 * uT * pv)
        if Q.dtype == torch.float16:
            tol += 2.0 ** -32 * v.abs().sum(1, keepdim=True) / total + 2.0 ** -25
        tolO[b] = tol.view(H, D)
        tolL[b] = (es.amax(-1, keepdim=True) + sums + R.EPS * (4 + (m + total.log()).abs())).view(H)
    return O, lse, tolO + 1e-37, tolL


def _check(dec, Q, cache, skip=()):
    O, lse, tO, tL = _exact(Q, cache, dec.max_len, skip)
    assert dec.status() == rkv.RKV_OK
    off = (dec.O.double() - O).abs()
    assert bool((off <= tO).all()), float((off / tO).max())
    inf = lse == -math.inf
    assert torch.equal(inf, dec.lse == -math.inf)
    assert bool(((dec.lse - lse).abs()[~inf] <= tL[~inf]).all()), float(((dec.lse - lse).abs() / tL)[~inf].max())


def _decoder(Q, cache, shared, top=None):
    B, H, D = Q.shape
    if top is None:
        top = int(max([0] + cache.lens.tolist()))
    dec = rkv.PrefixDecoder(H, cache.K.shape[1], D, top, B, Q.dtype, Q.device, num_groups=len(shared))
    dec.O.fill_(7.0)
    dec.lse.fill_(7.0)
    return dec


# (type, D, H, HK, page, layout, groups, alone)
CASES = [
    ("bf16", 128, 24, 8, 16, "hnd", [(1024, [1024 + i for i in range(10)])], []),
    ("bf16", 128, 24, 8, 16, "nhd", [(2048, [2048, 2100, 2049, 2560])], []),
    ("f16", 128, 16, 2, 32, "mixed", [(640, [640 + 7 * i for i in range(40)])], []),          # 320 rows
    ("bf16", 128, 8, 1, 16, "hnd", [(400, [400 + i for i in range(33)])], []),                # 264 rows, the last unit 8
    ("bf16", 128, 12, 4, 24, "hnd", [(480, [500] * 5), (96, [300, 96, 97]), (1200, [1300])], [5, 0, 700]),
    ("f16", 64, 24, 8, 8, "nhd", [(136, [140, 136, 300]), (512, [513] * 45)], [1]),
    ("bf16", 64, 8, 8, 1, "hnd", [(37, [40, 37, 50, 90])], []),                               # one token a page
    ("bf16", 96, 16, 2, 48, "hnd", [(1000, [1010 + i for i in range(9)])], []),               # shared tokens end inside a page
    ("f16", 80, 10, 5, 7, "mixed", [(333, [333, 400, 350]), (100, [90, 120, 0])], []),        # and shorter sequences
    ("bf16", 8, 16, 1, 16, "hnd", [(300, [301] * 3)], [20]),
    ("bf16", 128, 64, 1, 64, "hnd", [(3000, [3001, 3100])], []),                              # 64 heads of one KV head
    ("f16", 128, 3, 1, 16, "hnd", [(129, [130])] * 3, []),                                    # groups of one
    ("f32", 64, 8, 8, 24, "nhd", [(480, [500, 480, 700, 481, 490, 600])], []),
    ("f32", 128, 24, 8, 16, "hnd", [(512, [513] * 20), (1024, [1024, 1030])], [300]),
    ("f32", 256, 4, 2, 5, "hnd", [(123, [130, 125, 123, 3])], []),
    ("f32", 24, 3, 3, 5, "hnd", [(31, [31, 32])], []),
    ("bf16", 256, 16, 2, 16, "hnd", [(512, [520 + i for i in range(24)])], []),               # 192 rows of 256 columns
    ("f16", 248, 4, 2, 16, "hnd", [(700, [705] * 50), (300, [301] * 3)], []),
    ("bf16", 136, 40, 2, 16, "hnd", [(260, [270, 260])], []),
    ("f16", 128, 4, 2, 16, "hnd", [], [100, 0, 257]),                                          # no groups
    ("bf16", 128, 8, 4, 16, "hnd", [(0, [100, 50])], []),                                      # nothing shared
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])) + "-" + "+".join("%dx%d" % (len(x[1]), x[0]) for x in c[6]))
def test_prefix_decode_against_64_bits(case, cuda):
    kind, D, H, HK, page, layout, groups, alone = case
    cache, starts, shared = _setup(10, HK, D, page, groups, TYPES[kind], cuda, layout, alone)
    Q = _query(12, cache.batch, H, D, TYPES[kind], cuda)
    dec = _decoder(Q, cache, shared)
    got = dec(Q, cache, starts, shared)
    assert got is dec.O and got.dtype == TYPES[kind]
    _check(dec, Q, cache)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 300, 511, 640, 1023, 1025])
@pytest.mark.parametrize("kind,D,B", [("bf16", 128, 50), ("f16", 64, 30), ("bf16", 256, 30), ("f32", 128, 10)])
def test_every_end_of_a_tile(tokens, kind, D, B, cuda):
    dt = TYPES[kind]
    cache, starts, shared = _setup(20, 2, D, 16, [(tokens, [tokens + i % 3 for i in range(B)])], dt, cuda)
    Q = _query(21, B, 12, D, dt, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64), ("f16", 256), ("f32", 64)])
@pytest.mark.parametrize("B", [1, 2, 5, 6, 11, 21, 22, 43, 64, 90])
def test_every_number_of_rows(B, kind, D, cuda):
    """Rows on both sides of every unit's size: 6 B of a KV head."""
    dt = TYPES[kind]
    cache, starts, shared = _setup(22, 2, D, 32, [(448, [448 + i % 5 for i in range(B)])], dt, cuda)
    Q = _query(23, B, 12, D, dt, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 128), ("bf16", 256), ("f32", 128)])
def test_many_groups(kind, D, cuda):
    """More groups than lanes of a warp, some of them empty."""
    dt = TYPES[kind]
    g = torch.Generator().manual_seed(3)
    groups = []
    for i in range(75):
        p = int(torch.randint(1, 400, (1,), generator=g))
        groups.append((p, [p + j for j in range(int(torch.randint(0, 5, (1,), generator=g)))]))
    cache, starts, shared = _setup(30, 2, D, 16, groups, dt, cuda, alone=[9])
    Q = _query(31, cache.batch, 8, D, dt, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)


def test_large_scores_and_salient_keys(cuda):
    """Rows whose largest score moves late, far apart scores, and shared tokens
    that take nearly all of the weight, or none."""
    for kind, B in (("bf16", 60), ("f16", 60), ("f32", 4)):
        dt = TYPES[kind]
        cache, starts, shared = _setup(40, 2, 128, 16, [(3000, [3000 + 20 * (i % 4) for i in range(B)])], dt, cuda)
        order = cache.block_table[0, : 3000 // 16].long()
        cache.K[order] *= torch.linspace(0.1, 6.0, len(order), device=cuda).to(dt)[:, None, None, None]
        Q = _query(41, B, 12, 128, dt, cuda) * 4
        dec = _decoder(Q, cache, shared)
        dec(Q, cache, starts, shared)
        _check(dec, Q, cache)
        cache.K[order] *= -1
        dec(Q, cache, starts, shared)
        _check(dec, Q, cache)


@pytest.mark.parametrize("kind,B", [("bf16", 4), ("bf16", 60), ("f32", 4)])
def test_nothing_masked_is_read(kind, B, cuda):
    """NaN behind every sequence's end and in pages no sequence owns; page
    numbers behind the end, and for the shared tokens of all but the first
    sequence, that lie outside the pool."""
    dt, page = TYPES[kind], 16
    lens = [200 + i for i in range(B)]
    lens[0], lens[-1] = 30, 0  # the first holds too few tokens to be read through, the last is idle
    cache, starts, shared = _setup(50, 2, 128, page, [(160, lens)], dt, cuda)
    Q = _query(51, B, 6, 128, dt, cuda)
    want = _decoder(Q, cache, shared, 256)
    want(Q, cache, starts, shared)
    _check(want, Q, cache)
    keep = torch.zeros((cache.K.shape[0], page), dtype=torch.bool, device=cuda)
    for b, n in enumerate(lens):
        t = torch.arange(n, device=cuda)
        keep[cache.block_table[b].long()[t // page], t % page] = True
    cache.K.masked_fill_(~keep[:, None, :, None], math.nan)
    cache.V.masked_fill_(~keep[:, None, :, None], math.inf)
    for b, n in enumerate(lens):
        cache.block_table[b, -(-n // page):] = -1 if b % 2 else 10 ** 6
        if b > 1 and n:
            cache.block_table[b, : 160 // page] = 2 ** 31 - 1
    got = _decoder(Q, cache, shared, 256)
    got(Q, cache, starts, shared)
    assert torch.equal(got.O, want.O) and torch.equal(got.lse, want.lse)


@pytest.mark.parametrize("kind,B", [("f16", 3), ("bf16", 50), ("f32", 3)])
def test_pages_outside_the_pool_are_left_out(kind, B, cuda):
    dt, page, n = TYPES[kind], 16, 300
    cache, starts, shared = _setup(60, 2, 64, page, [(256, [n] * B)], dt, cuda)
    cache.block_table[:, 3] = -1
    cache.block_table[:, 8:16] = cache.K.shape[0]  # a whole tile
    cache.block_table[1, 17] = 2 ** 31 - 1
    skip = {(b, t) for b in range(B) for t in list(range(48, 64)) + list(range(128, 256))} | {(1, t) for t in range(272, 288)}
    Q = _query(61, B, 6, 64, dt, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache, skip)
    cache.block_table.fill_(-1)  # nothing left
    dec(Q, cache, starts, shared)
    assert bool((dec.O == 0).all()) and bool((dec.lse == -math.inf).all()) and dec.status() == rkv.RKV_OK


@pytest.mark.parametrize("kind,B", [("bf16", 2), ("bf16", 50), ("f32", 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_values_stay_where_they_are(kind, B, bad, cuda):
    """In a shared row of V: in its column of its KV head's outputs of the
    group, nowhere else.  In a shared row of K: in its KV head's outputs of the
    group."""
    dt, D, H, HK = TYPES[kind], 128, 6, 3
    cache, starts, shared = _setup(70, HK, D, 16, [(400, [420] * B), (64, [70, 80])], dt, cuda)
    Q = _query(71, B + 2, H, D, dt, cuda)
    dec, ref = _decoder(Q, cache, shared), _decoder(Q, cache, shared)
    ref(Q, cache, starts, shared)
    at, row = cache.block_table[0, 20].long(), 7
    cache.V[at, 1, row, 5] = bad
    dec(Q, cache, starts, shared)
    hit = torch.zeros_like(dec.O, dtype=torch.bool)
    hit[:B, 2:4, 5] = True
    assert not bool(dec.O[hit].isfinite().any()) and torch.equal(dec.O[~hit], ref.O[~hit]) and torch.equal(dec.lse, ref.lse)
    cache.V[at, 1, row, 5] = 1.0
    ref(Q, cache, starts, shared)
    cache.K[at, 1, row, 5] = bad
    dec(Q, cache, starts, shared)
    hit[:B, 2:4] = True
    assert torch.equal(dec.O[~hit], ref.O[~hit])
    if not math.isfinite(bad) and bad != bad:
        assert not bool(dec.O[hit].isfinite().any())


def test_groups_are_clamped(cuda):
    """Starts outside the batch, shared tokens beyond max_len, the table and
    below 0; lengths that are clamped."""
    dt, B = torch.bfloat16, 6
    cache, starts, shared = _setup(80, 2, 64, 16, [(64, [70, 80, 64]), (32, [40, 50, 60])], dt, cuda)
    Q = _query(81, B, 4, 64, dt, cuda)
    dec = _decoder(Q, cache, shared)
    for s, t in (([-5, 3, 900], [64, 32]), ([0, 3, 6], [10 ** 9, 2 ** 31 - 1]), ([0, 3, 6], [-3, -2 ** 31]), ([9, 9, 9], [5, 5]),
                 ([0, 0, 3], [7, 64]), ([6, 3, 0], [64, 64])):
        dec(Q, cache, torch.tensor(s, dtype=torch.int32, device=cuda), torch.tensor(t, dtype=torch.int32, device=cuda))
        _check(dec, Q, cache)
    cache.lens.copy_(torch.tensor([1000, 70, 64, -7, 50, 60], dtype=torch.int32))
    few = _decoder(Q, cache, shared, 66)
    few(Q, cache, starts, shared)
    cache.lens.copy_(torch.tensor([66, 66, 64, 0, 50, 60], dtype=torch.int32))
    _check(few, Q, cache)


@pytest.mark.parametrize("D,B", [(128, 40), (128, 3), (256, 20)])
def test_offsets_past_32_bits(D, B, cuda):
    """A pool of more than 2^32 bytes whose last pages are shared."""
    HK, page = 4, 128
    pages = (1 << 32) // (HK * page * D * 2) + 40
    K = torch.empty((pages, HK, page, D), dtype=torch.bfloat16, device=cuda)
    tab = torch.tensor([[pages - 1, 0, pages - 3, 3 + b] for b in range(B)], dtype=torch.int32, device=cuda)
    for p in set(tab.view(-1).tolist()):
        K[p] = torch.randn((HK, page, D), device=cuda).to(torch.bfloat16)
    cache = rkv.PagedCache(K, K, tab, torch.tensor([384 + b for b in range(B)], dtype=torch.int32, device=cuda))
    starts, shared = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, B], [384]))
    Q = _query(91, B, 12, D, torch.bfloat16, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)


@pytest.mark.parametrize("kind,D,B", [("bf16", 128, 40), ("f16", 64, 3), ("f32", 128, 7), ("bf16", 256, 30)])
def test_repeats_bit_for_bit_and_in_a_graph(kind, D, B, cuda):
    """The same call twice, the call in a captured graph replayed over other
    lengths, groups and queries, and two objects on two streams."""
    dt = TYPES[kind]
    cache, starts, shared = _setup(100, 2, D, 16, [(1600, [1700 + i for i in range(B - 1)]), (800, [900])], dt, cuda)
    Q = _query(101, B, 12, D, dt, cuda)
    dec = _decoder(Q, cache, shared)
    dec(Q, cache, starts, shared)
    first, lse = dec.O.clone(), dec.lse.clone()
    dec.O.zero_()
    dec(Q, cache, starts, shared)
    assert torch.equal(dec.O, first) and torch.equal(dec.lse, lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec(Q, cache, starts, shared)
    for cut, seed in ((0, 101), (900, 102), (1690, 103)):
        cache.lens.copy_(torch.tensor([max(0, 1700 + i - cut) for i in range(B - 1)] + [850], dtype=torch.int32))
        shared.copy_(torch.tensor([max(1, 1600 - cut), 33], dtype=torch.int32))
        Q.copy_(_query(seed, B, 12, D, dt, cuda))
        g.replay()
        torch.cuda.synchronize()
        _check(dec, Q, cache)
    other, want = _decoder(Q, cache, shared), dec.O.clone()
    torch.cuda.synchronize()
    for s, d in zip([torch.cuda.Stream() for _ in range(2)], (dec, other)):
        for _ in range(3):
            d(Q, cache, starts, shared, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(dec.O, want)
    _check(other, Q, cache)


def test_calls_one_behind_the_other_share_a_workspace(cuda):
    """Calls of one object over other groups at once behind each other."""
    dt, B = torch.bfloat16, 48
    cache, starts, shared = _setup(110, 2, 128, 16, [(1024, [1024 + i for i in range(B)])], dt, cuda)
    Q = [_query(111 + i, B, 12, 128, dt, cuda) for i in range(4)]
    cut = [torch.tensor([n], dtype=torch.int32, device=cuda) for n in (1024, 100, 513, 1)]
    ref = []
    for q, c in zip(Q, cut):
        d = _decoder(q, cache, shared)
        d(q, cache, starts, c)
        _check(d, q, cache)
        ref.append(d.O.clone())
    dec, got = _decoder(Q[0], cache, shared), []
    for _ in range(5):
        got = [dec(q, cache, starts, c).clone() for q, c in zip(Q, cut)]
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_buffers_outlive_their_object_while_a_call_on_another_stream_runs(cuda):
    cache, starts, shared = _setup(120, 2, 64, 16, [(160, [180, 170, 200])], torch.bfloat16, cuda)
    Q = _query(121, 3, 4, 64, torch.bfloat16, cuda)
    s = torch.cuda.Stream()
    for cycles in (1000, 200_000_000):  # first to load and allocate; then about 100 ms
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(cycles)
        dec = rkv.PrefixDecoder(4, 2, 64, 200, 3, torch.bfloat16, cuda)
        dec(Q, cache, starts, shared, stream=s.cuda_stream)
        mine = [(t.data_ptr(), t.numel() * t.element_size()) for t in (dec.ws, dec.O, dec.lse)]
        del dec
        new = [torch.empty(size, dtype=torch.uint8, device=cuda) for _, size in mine for _ in range(4)]
        busy = not s.query()
    assert busy, "the call ended too early to show anything"
    for t in new:
        for at, size in mine:
            assert t.data_ptr() + t.numel() <= at or at + size <= t.data_ptr()
    torch.cuda.synchronize()


def test_empty_calls(cuda):
    K, V = R.pool(8, 6, 2, 16, 64, torch.bfloat16, cuda)
    c = rkv.PagedCache(K, V, torch.empty((0, 4), dtype=torch.int32, device=cuda), torch.empty(0, dtype=torch.int32, device=cuda))
    z = torch.zeros(2, dtype=torch.int32, device=cuda)
    dec = rkv.PrefixDecoder(4, 2, 64, 50, 0, torch.bfloat16, cuda)
    assert dec.status() == rkv.RKV_OK
    assert dec(torch.empty((0, 4, 64), dtype=torch.bfloat16, device=cuda), c, z, z[:1]).shape == (0, 4, 64)
    assert dec.status() == rkv.RKV_OK
    # sequences without a token, and a cache of no pages at all
    c = rkv.PagedCache(K, V, torch.zeros((3, 4), dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda))
    dec = rkv.PrefixDecoder(4, 2, 64, 0, 3, torch.bfloat16, cuda)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=cuda)
    for cache in (c, rkv.PagedCache(K[:0], V[:0], torch.zeros((3, 4), dtype=torch.int32, device=cuda),
                                    torch.full((3,), 9, dtype=torch.int32, device=cuda))):
        dec.O.fill_(7.0)
        dec(q, cache, torch.tensor([0, 3], dtype=torch.int32, device=cuda), torch.tensor([20], dtype=torch.int32, device=cuda))
        assert bool((dec.O == 0).all()) and bool((dec.lse == -math.inf).all()) and dec.status() == rkv.RKV_OK


def test_refused_calls(cuda):
    cache, starts, shared = _setup(130, 2, 64, 16, [(160, [180, 170])], torch.bfloat16, cuda)
    Q = _query(131, 2, 4, 64, torch.bfloat16, cuda)
    dec = _decoder(Q, cache, shared)
    for bad in (dict(Q=Q.float()), dict(Q=Q[:1]), dict(Q=Q.transpose(0, 1)), dict(group_starts=starts[:1]), dict(group_tokens=starts),
                dict(group_starts=starts.long()), dict(group_tokens=shared.cpu())):
        with pytest.raises((ValueError, TypeError)):
            dec(**{**dict(Q=Q, cache=cache, group_starts=starts, group_tokens=shared), **bad})
    with pytest.raises(ValueError):  # the output's type is the cache's
        rkv.PrefixDecoder(4, 2, 64, 200, 2, torch.float16, cuda)(Q, cache, starts, shared)
    with pytest.raises(rkv.RkvError):
        rkv.PrefixDecoder(4, 3, 64, 200, 2, torch.float16, cuda)
    assert bool((dec.O == 7.0).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_batches_without_tokens_or_pages(D, cuda):
    B = 40
    K, V = R.pool(8, 6, 2, 16, D, torch.bfloat16, cuda)
    q = _query(9, B, 4, D, torch.bfloat16, cuda)
    starts, shared = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, B], [20]))
    tab = torch.zeros((B, 4), dtype=torch.int32, device=cuda)
    for cache, top in ((rkv.PagedCache(K, V, tab, torch.zeros(B, dtype=torch.int32, device=cuda)), 60),
                       (rkv.PagedCache(K, V, tab, torch.full((B,), 30, dtype=torch.int32, device=cuda)), 0),
                       (rkv.PagedCache(K[:0], V[:0], tab, torch.full((B,), 30, dtype=torch.int32, device=cuda)), 60),
                       (rkv.PagedCache(K, V, tab[:, :0], torch.full((B,), 30, dtype=torch.int32, device=cuda)), 60)):
        dec = _decoder(q, cache, shared, top)
        dec(q, cache, starts, shared)
        assert dec.status() == rkv.RKV_OK
        assert bool((dec.O == 0).all()) and bool((dec.lse == -math.inf).all())


@pytest.mark.parametrize("seed", range(36))
def test_random_batches(seed, cuda):
    """Groups, lengths, pages, heads and layouts drawn together."""
    import random
    r = random.Random(seed)
    kind = r.choice(["bf16", "f16", "f32"])
    D = r.choice([8, 32, 64, 72, 96, 128, 128, 136, 200, 256])
    HK, G = r.choice([1, 2, 3]), r.choice([1, 2, 5, 8, 12])
    page, layout = r.choice([1, 3, 8, 16, 24, 64, 128, 200]), r.choice(["hnd", "nhd", "mixed"])
    groups = []
    for _ in range(r.randint(1, 5)):
        p = r.choice([0, r.randint(1, 300), r.randint(100, 900)])
        groups.append((p, [r.choice([p, p + r.randint(0, 400), p + 1, max(0, p - r.randint(0, 60)), 0]) for _ in range(r.randint(0, 20))]))
    alone = [r.randint(0, 300) for _ in range(r.randint(0, 3))]
    if not any(x[1] for x in groups) and not alone:
        alone = [5]
    dt = TYPES[kind]
    cache, starts, shared = _setup(200 + seed, HK, D, page, groups, dt, cuda, layout, alone)
    Q = _query(300 + seed, cache.batch, HK * G, D, dt, cuda)
    dec = _decoder(Q, cache, shared, max(1, int(cache.lens.max())) + r.choice([0, 100, 5000]))
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)
