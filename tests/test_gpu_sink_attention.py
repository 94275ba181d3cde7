"""Prefill attention with a sliding window and sinks on the GPU, against the
formula in 64 bits (tests/pagedref.py), and a prompt taken through it, the
window eviction and the paged decode."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(seed, B, H, HK, Lq, Lk, D, dtype, dev, token_major=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    if token_major:  # a fused projection's buffer [B, tokens, H + 2 HK, D]
        buf = torch.randn((B, Lk, H + 2 * HK, D), generator=g, device=dev).to(dtype).transpose(1, 2)
        return buf[:, :H, Lk - Lq:], buf[:, H:H + HK], buf[:, H + HK:]
    mk = lambda h, n: torch.randn((B, h, n, D), generator=g, device=dev).to(dtype)  # noqa: E731
    return mk(H, Lq), mk(HK, Lk), mk(HK, Lk)


def _check(Q, K, V, sinks, window, lens, out, lse, O0, lse0):
    O, L, tO, tL = R.sink_attention(Q, K, V, sinks, window, lens)
    real = ~L.isnan()
    d = (out.double() - O).abs()[real]
    assert bool((d <= tO[real]).all()), float((d / tO[real]).max())
    assert bool(((lse - L).abs()[real] <= tL[real]).all())
    assert torch.equal(out[~real], O0[~real]) and torch.equal(lse[~real], lse0[~real])


CASES = [
    # type, D, H, HK, len_q, len_k, sinks, window, lens
    ("bf16", 128, 24, 8, 512, 512, 0, 0, None),
    ("bf16", 128, 6, 2, 700, 700, 4, 128, None),
    ("bf16", 128, 4, 4, 1, 1, 0, 0, None),
    ("bf16", 128, 4, 2, 1, 513, 2, 100, None),             # a single query behind a prefix
    ("f16", 128, 8, 2, 257, 1030, 0, 0, None),
    ("f16", 64, 8, 2, 1289, 1537, 4, 250, [1537, 900, 249, 248, 247, 0]),
    ("bf16", 64, 4, 1, 130, 130, 0, 1, None),              # each query sees itself alone
    ("bf16", 128, 4, 1, 300, 300, 300, 1, None),           # sinks over all
    ("bf16", 128, 2, 1, 600, 600, 200, 3, [600, 129, 128, 127, 1]),
    ("f32", 128, 6, 2, 200, 333, 4, 64, [333, 200, 134, 133]),
    ("f32", 64, 8, 8, 129, 129, 0, 0, None),
    ("f32", 256, 2, 1, 70, 100, 1, 20, None),
    ("bf16", 256, 4, 2, 200, 260, 4, 100, [260, 100]),
    ("f16", 96, 4, 2, 150, 150, 0, 77, None),
    ("bf16", 72, 3, 3, 140, 300, 5, 60, [300, 161]),
    ("f16", 8, 2, 1, 65, 65, 0, 0, None),
    ("f16", 120, 2, 2, 129, 1000, 0, 300, None),
    ("bf16", 200, 2, 1, 129, 129, 0, 0, None),
    ("bf16", 128, 2, 2, 2050, 2050, 64, 512, None),
    ("f16", 128, 1, 1, 128, 4097, 130, 1000, [4000]),
    ("f16", 256, 3, 1, 1100, 1100, 4, 500, [1100, 700, 64, 63, 0]),
    ("bf16", 136, 24, 8, 700, 900, 0, 0, None),            # more units than SMs
    ("f16", 192, 2, 2, 65, 2000, 70, 333, [2000, 1999]),
    # few queries over many keys: the keys are taken in parts
    ("bf16", 128, 8, 2, 64, 8000, 0, 0, None),
    ("bf16", 128, 3, 1, 300, 9000, 4, 2500, [9000, 8701, 8700, 3]),
    ("f16", 64, 4, 4, 5, 7001, 600, 40, [7001, 7000, 6997, 6996]),
    ("f32", 128, 2, 1, 33, 6000, 0, 0, [6000, 5970]),
    ("f32", 256, 2, 2, 10, 5000, 130, 1000, None),
    ("bf16", 256, 4, 1, 20, 6100, 0, 0, [6100, 6085]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, (c[0], "d%d" % c[1]) + c[2:8])))
@pytest.mark.parametrize("token_major", [False, True])
def test_against_64_bits(case, token_major, cuda):
    kind, D, H, HK, Lq, Lk, sinks, window, lens = case
    dt, B = TYPES[kind], len(lens) if lens else 2
    Q, K, V = _inputs(7, B, H, HK, Lq, Lk, D, dt, cuda, token_major)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda) if lens else None
    if lens:  # padding is never read
        K, V = (x.clone() if not token_major else x for x in (K, V))
        for b, n in enumerate(lens):
            K[b, :, n:], V[b, :, n:] = math.nan, math.inf
    out = torch.full((B, Lq, H, D), 3.0, device=cuda).to(dt).transpose(1, 2) if token_major else torch.full_like(Q, 3.0)
    lse = torch.full((B, H, Lq), 5.0, device=cuda)
    O0, lse0 = out.clone(), lse.clone()
    att = rkv.SinkAttention(sinks=sinks, window=window, device=cuda)
    att(Q, K, V, lens=lt, out=out, lse=lse)
    assert att.status() == 0
    _check(Q, K, V, sinks, window, lens, out, lse, O0, lse0)


@pytest.mark.parametrize("D,window", [(64, 0), (128, 70), (256, 0)])
def test_many_ragged_sequences(D, window, cuda):
    """Several times as many items as SMs, of very different lengths and some
    without a row, an odd number of query tiles per KV head; the same bits when
    the calls run on two streams at once."""
    B, H, HK, n = 60, 6, 2, 300
    Q, K, V = _inputs(31, B, H, HK, n, n, D, torch.bfloat16, cuda)
    lens = [(37 * b * b + 11 * b) % (n + 1) if b % 7 else 0 for b in range(B)]
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    runs = [(rkv.SinkAttention(sinks=2, window=window, device=cuda), torch.full_like(Q, 3.0),
             torch.full((B, H, n), 5.0, device=cuda), torch.cuda.Stream()) for _ in range(2)]
    O0, lse0 = runs[0][1].clone(), runs[0][2].clone()
    torch.cuda.synchronize()
    for _ in range(3):
        for att, out, lse, st in runs:
            att(Q, K, V, lens=lt, out=out, lse=lse, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(att.status() == 0 for att, *_ in runs)
    _check(Q, K, V, 2, window, lens, runs[0][1], runs[0][2], O0, lse0)
    assert torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])


def test_large_scores(cuda):
    """Scores far apart, largest late or early in the row."""
    Q, K, V = _inputs(8, 1, 4, 2, 400, 400, 128, torch.bfloat16, cuda)
    Q = Q * 4
    for order in (torch.linspace(0.1, 8, 400), torch.linspace(8, 0.1, 400)):
        Ks = (K.float() * order.to(cuda)[None, None, :, None]).to(torch.bfloat16)
        lse, out = torch.zeros((1, 4, 400), device=cuda), torch.zeros_like(Q)
        rkv.SinkAttention(device=cuda)(Q, Ks, V, out=out, lse=lse)
        _check(Q, Ks, V, 0, 0, None, out, lse, out, lse)


def test_lengths_beyond_the_keys_are_clamped(cuda):
    Q, K, V = _inputs(9, 3, 2, 1, 100, 140, 64, torch.float16, cuda)
    out, lse = torch.zeros_like(Q), torch.zeros((3, 2, 100), device=cuda)
    rkv.SinkAttention(device=cuda)(Q, K, V, lens=torch.tensor([10 ** 9, 100, -4], dtype=torch.int32, device=cuda), out=out, lse=lse)
    _check(Q, K, V, 0, 0, [140, 100, 0], out, lse, torch.zeros_like(out), torch.zeros_like(lse))


def test_repeats_and_graph(cuda):
    """Bit for bit again, captured and replayed over other inputs, on two
    streams with a workspace each."""
    Q, K, V = _inputs(11, 2, 8, 2, 600, 700, 128, torch.bfloat16, cuda)
    lens = torch.tensor([700, 300], dtype=torch.int32, device=cuda)
    att = rkv.SinkAttention(sinks=4, window=200, device=cuda)
    out, lse = torch.zeros_like(Q), torch.zeros((2, 8, 600), device=cuda)
    att(Q, K, V, lens=lens, out=out, lse=lse)
    first = out.clone()
    out.zero_()
    att(Q, K, V, lens=lens, out=out, lse=lse)
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        att(Q, K, V, lens=lens, out=out, lse=lse)
    Q2, K2, V2 = _inputs(12, 2, 8, 2, 600, 700, 128, torch.bfloat16, cuda)
    for t, s in ((Q, Q2), (K, K2), (V, V2), (lens, torch.tensor([450, 700], dtype=torch.int32))):
        t.copy_(s)
    out.zero_()
    lse.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert att.status() == 0
    _check(Q, K, V, 4, 200, lens.tolist(), out, lse, torch.zeros_like(out), torch.zeros_like(lse))
    want = out.clone()
    # a larger call makes the workspace grow; the captured one still has its own
    Ql, Kl, Vl = _inputs(13, 1, 8, 2, 60, 9000, 128, torch.bfloat16, cuda)
    att(Ql, Kl, Vl)
    junk = torch.full((1 << 22,), math.nan, device=cuda)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del junk
    both = [(rkv.SinkAttention(sinks=4, window=200, device=cuda), torch.zeros_like(Q), torch.cuda.Stream()) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for a, o, s in both:
            a(Q, K, V, lens=lens, out=o, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, o, _ in both)


def test_output_of_a_call_on_another_stream(cuda):
    """What a call allocates is filled on its own stream: work queued on the
    current one does not come behind the attention."""
    Q, K, V = _inputs(21, 1, 4, 2, 200, 200, 64, torch.bfloat16, cuda)
    att, s = rkv.SinkAttention(device=cuda), torch.cuda.Stream()
    want = att(Q, K, V)
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)  # about 25 ms
    out = att(Q, K, V, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_prompt_through_prefill_eviction_and_decode(cuda):
    """A prompt's attention, stage 1 on its own Q and K, the kept rows put into
    pages, and the next token decoded over them: the decode equals plain
    attention over the kept rows."""
    H, HK, D, n, budget, page = 6, 2, 128, 600, 160, 16
    dt = torch.bfloat16
    Q, K, V = _inputs(15, 1, H, HK, n, n, D, dt, cuda)
    rkv.SinkAttention(sinks=4, window=256, device=cuda)(Q, K, V)
    cfg = rkv.RocketConfig(num_heads=H, num_heads_kv=HK, dim_head=D, prompt_budget=budget)
    kept, cnt = rkv.Evictor(cfg, n, n, 1, rkv.BF16, cuda)(Q, K)
    m = int(cnt[0])
    t = kept[0, :m].long()
    per = -(-(m + 1) // page)
    Kp, Vp = R.pool(16, per + 2, HK, page, D, dt, cuda)
    lens = torch.tensor([m], dtype=torch.int32, device=cuda)
    cache = rkv.PagedCache(Kp, Vp, R.table(17, 1, per, per + 2, cuda), lens)
    rkv.paged_append(cache, K[:, :, t].transpose(1, 2), V[:, :, t].transpose(1, 2))
    lens += 1
    g = torch.Generator(device=cuda).manual_seed(18)
    k1, v1, q1 = (torch.randn((1, h, D), generator=g, device=cuda).to(dt) for h in (HK, HK, H))
    rkv.paged_append(cache, k1, v1)
    dec = rkv.PagedDecoder(H, HK, D, m + 1, 1, cuda)
    dec(q1, cache)
    for h in range(H):
        kk = torch.cat((K[0, h // 3, t], k1[0, h // 3][None])).double()
        vv = torch.cat((V[0, h // 3, t], v1[0, h // 3][None])).double()
        want = torch.softmax(q1[0, h].double() @ kk.T / math.sqrt(D), 0) @ vv
        assert float((dec.O[0, h] - want).abs().max()) < 1e-4
