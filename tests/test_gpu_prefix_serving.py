"""The rotated rows, the paged cache and the shared-prefix decode together, as a
server uses them: a prompt is turned, attended and put into pages that several
answers share, and each step turns and appends its rows and attends them."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv
from test_gpu_prefix import _exact
from test_gpu_rotary import _turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,B,axes", [("bf16", 3, 1), ("f16", 12, 3), ("f32", 2, 1)])
def test_answers_to_one_prompt(kind, B, axes, cuda):
    """Against attention in 64 bits over the rows that the cache holds, and
    the held rows against the formula."""
    dt = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]
    H, HK, D, page, n, steps = 12, 4, 64, 16, 336, 5
    g = torch.Generator(device=cuda).manual_seed(4)
    fr = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    ax = None if axes == 1 else torch.arange(D // 2) * axes // (D // 2)
    rotary = rkv.Rotary(fr, D, axes=ax, num_axes=axes, device=cuda)
    shared, own = n // page, -(-steps // page)
    K, V = R.pool(5, shared + B * own + 2, HK, page, D, dt, cuda)
    order = torch.randperm(K.shape[0], generator=torch.Generator().manual_seed(6)).tolist()
    prompt = order[:shared]
    rows = [prompt + order[shared + b * own: shared + (b + 1) * own] for b in range(B)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731

    # the prompt: one sequence's rows, turned, attended and put into the shared pages
    qkv = torch.randn((1, n, H + 2 * HK, D), generator=g, device=cuda).to(dt)
    q, k, v = (x.transpose(1, 2) for x in qkv.split([H, HK, HK], dim=2))
    pos = torch.stack([torch.arange(n, device=cuda) // (a + 1) for a in range(axes)])[:, None].to(torch.int32).contiguous()
    want, tol = _turn(k, pos, fr, ax, False)
    qr, kr = rkv.rotate(q, k, pos, rotary, q_out=q, k_out=k)  # in place: k stays laid out as v
    assert bool(((kr.double() - want).abs() <= tol).all())
    O = rkv.SinkAttention(device=cuda)(qr, kr, v)
    oO, _, tO, _ = R.sink_attention(qr, kr, v, 0, 0)
    assert bool(((O - oO).abs() <= tO).all())
    rkv.paged_append(rkv.PagedCache(K, V, i32([prompt]), i32([n])), kr.transpose(1, 2), v.transpose(1, 2))

    # the answers
    lens, starts, tokens = i32([n] * B), i32([0, B]), i32([n])
    cache = rkv.PagedCache(K, V, i32(rows), lens)
    dec = rkv.PrefixDecoder(H, HK, D, n + steps, B, dt, cuda)
    plain = rkv.PagedDecoder(H, HK, D, n + steps, B, cuda)
    q_out = torch.empty((B, H, D), dtype=dt, device=cuda)
    new, at = torch.empty((B, H + 2 * HK, D), dtype=dt, device=cuda), torch.empty((axes, B), dtype=torch.int32, device=cuda)

    def step():
        qn, kn, vn = new.split([H, HK, HK], dim=1)
        rkv.paged_append_rotated(cache, kn, vn, rotary, q=qn, q_out=q_out, positions=at[:, :, None])
        dec(q_out, cache, starts, tokens)

    graph = None
    for i in range(steps):
        lens.add_(1)
        new.copy_(torch.randn(new.shape, generator=g, device=cuda).to(dt))
        at.copy_(torch.stack([torch.full((B,), n // (a + 1) + 7 * i, device=cuda) for a in range(axes)]))
        if graph is None:
            step()  # loads what a capture must not
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay()
        torch.cuda.synchronize()
        qw, qt = _turn(new[:, :H, None], at[:, :, None], fr, ax, False)
        assert bool(((q_out[:, :, None].double() - qw).abs() <= qt).all())
        kw, kt = _turn(new[:, H: H + HK, None], at[:, :, None], fr, ax, False)
        t = n + i
        page_of = cache.block_table[:, t // page].long()
        assert bool(((K[page_of, :, t % page].double() - kw[:, :, 0]).abs() <= kt[:, :, 0]).all())
        assert torch.equal(V[page_of, :, t % page], new[:, H + HK:])
        O, lse, tO, tL = _exact(q_out, cache, n + steps)
        assert bool(((dec.O.double() - O).abs() <= tO).all()) and bool(((dec.lse - lse).abs() <= tL).all())
        assert dec.status() == rkv.RKV_OK
        plain(q_out, cache)
        assert bool(((plain.O.double() - O).abs() <= tO).all())
    assert int(lens[0]) == n + steps and not math.isnan(float(dec.O.float().sum()))


def test_two_decoders_at_once(cuda):
    """An object each, on two streams, beside an append of other sequences."""
    from test_gpu_prefix import _query, _setup
    cache, starts, tokens = _setup(7, 2, 128, 16, [(1024, [1024 + 3 * i for i in range(30)])], torch.bfloat16, cuda)
    Q = [_query(8 + i, 30, 12, 128, torch.bfloat16, cuda) for i in range(2)]
    decs = [rkv.PrefixDecoder(12, 2, 128, 1200, 30, torch.bfloat16, cuda) for _ in range(2)]
    want = [d(q, cache, starts, tokens).clone() for d, q in zip(decs, Q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, q, s in zip(decs, Q, streams):
            d(q, cache, starts, tokens, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(d.O, w) and d.status() == rkv.RKV_OK for d, w in zip(decs, want))
