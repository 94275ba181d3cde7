"""Calls of the sink-window prefill attention one after the other and by one
object: workspaces, the error word, sequences without rows, weights far below
their row's largest."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu


def _inputs(seed, B, H, HK, Lq, Lk, D, dtype, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda h, n: torch.randn((B, h, n, D), generator=g, device=dev).to(dtype)  # noqa: E731
    return mk(H, Lq), mk(HK, Lk), mk(HK, Lk)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 256), (torch.float32, 64)])
def test_nothing_to_join_then_a_call_on_the_same_workspace(dtype, D, cuda):
    """Keys in parts and every query behind its sequence's end: nothing is
    written, and calls behind it on the stream find the workspace free."""
    B, H, HK, Lq, Lk = 2, 4, 2, 40, 5000
    Q, K, V = _inputs(1, B, H, HK, Lq, Lk, D, dtype, cuda)
    none = torch.tensor([Lk - Lq, 17], dtype=torch.int32, device=cuda)
    lens = torch.tensor([Lk, Lk - 11], dtype=torch.int32, device=cuda)
    att = rkv.SinkAttention(sinks=4, device=cuda)
    want, want_lse = torch.full_like(Q, 3.0), torch.full((B, H, Lq), 5.0, device=cuda)
    att(Q, K, V, lens=lens, out=want, lse=want_lse)
    O, L, tO, tL = R.sink_attention(Q, K, V, 4, 0, lens.tolist())
    real = ~L.isnan()
    assert bool(((want.double() - O).abs()[real] <= tO[real]).all()) and bool(((want_lse - L).abs()[real] <= tL[real]).all())
    for _ in range(20):
        out, lse = torch.full_like(Q, 3.0), torch.full((B, H, Lq), 5.0, device=cuda)
        empty, empty_lse = torch.full_like(Q, 3.0), torch.full((B, H, Lq), 5.0, device=cuda)
        att(Q, K, V, lens=none, out=empty, lse=empty_lse)
        att(Q, K, V, lens=lens, out=out, lse=lse)
        assert bool((empty == 3.0).all()) and bool((empty_lse == 5.0).all())
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert att.status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,q0,k0", [(64, 12.0, 12.0), (128, 12.0, 17.0), (256, 16.0, 18.0)])
def test_many_small_weights_count(dtype, D, q0, k0, cuda):
    """One key 18 above all others, whose V is 0: the output is what 40000
    weights of e^-18 = 2^-26 add up to.  Against the formula in 64 bits: such a
    weight as an fp16 number 2^7 larger is off by half of its fixed step, 2^-32,
    or relative by half a step of the type; then the output by half a step
    (fp32's own errors, 2^-24 a term at the most, are below both)."""
    H, Lq, Lk = 40, 300, 40000  # every SM has queries, so the keys stay in one part
    Q, K = torch.zeros((1, H, Lq, D), dtype=dtype, device=cuda), torch.zeros((1, H, Lk, D), dtype=dtype, device=cuda)
    Q[..., 0], K[:, :, 0, 0] = q0, k0
    g = torch.Generator(device=cuda).manual_seed(3)
    V = (1 + torch.rand((1, H, Lk, D), generator=g, device=cuda)).to(dtype)
    V[:, :, 0] = 0
    out, lse = torch.zeros_like(Q), torch.zeros((1, H, Lq), device=cuda)
    att = rkv.SinkAttention(device=cuda)
    att(Q, K, V, out=out, lse=lse)
    assert att.status() == 0
    s, u = q0 * k0 / math.sqrt(D), R.unit(dtype)
    w = math.exp(-s)
    p = torch.arange(Lk - Lq, Lk, device=cuda, dtype=torch.float64)
    total = 1 + p * w
    for h in range(H):
        add = V[0, h].double().cumsum(0)[Lk - Lq:]
        want = add * w / total[:, None]
        fixed = 2.0 ** -32 * p[:, None] * 2 if dtype == torch.float16 else 0.0  # V < 2
        sums = R.EPS * (625 + 16 * s)
        tol = want * (2 * u + sums) + fixed
        off = float(((out[0, h] - want).abs() / tol).max())
        assert off <= 1, (h, off)
    # the weights' sum is rounded once a tile, and with equal terms always the same way: up to 625 tiles of 64 keys,
    # 625 * 2^-24 of it; the exponent's largest term and lse itself a few times
    off = float((lse[0].double() - s - total.log()).abs().max())
    assert off <= R.EPS * (625 + 8 * s), off


def test_status_of_an_object_that_has_not_run(cuda):
    """No error word is read that no call has written: neither of a new
    object, in memory that held something else, nor after calls without work."""
    for _ in range(8):  # blocks of the size a workspace has, given back full of ones
        junk = [torch.full((256,), 255, dtype=torch.uint8, device=cuda) for _ in range(64)]
        del junk
        att = rkv.SinkAttention(device=cuda)
        assert att.status() == 0
        Q, K, V = _inputs(5, 0, 2, 1, 8, 8, 64, torch.bfloat16, cuda)
        att(Q, K, V)
        Q, K, V = _inputs(5, 1, 2, 1, 0, 8, 64, torch.bfloat16, cuda)
        att(Q, K, V)
        assert att.status() == 0


def test_status_of_a_call_whose_workspace_was_outgrown(cuda):
    """An error that a call recorded is found after the workspace has grown,
    once, and whatever the other calls recorded."""
    att = rkv.SinkAttention(device=cuda)
    Q, K, V = _inputs(6, 1, 2, 1, 8, 8, 64, torch.bfloat16, cuda)
    att(Q, K, V)
    first = att.ws
    att(*_inputs(6, 1, 2, 1, 8, 5000, 64, torch.bfloat16, cuda))
    assert att.ws is not first and att.status() == 0
    first[:4].view(torch.int32).fill_(rkv.RKV_ERR_DEVICE_TIMEOUT)  # as the kernel records it
    assert att.status() == rkv.RKV_ERR_DEVICE_TIMEOUT
    assert att.status() == 0


def test_a_fresh_output_is_filled_only_where_rows_stay_unwritten(cuda, monkeypatch):
    """Zeros behind the ends of padded sequences; without lens every row is
    written and nothing else is launched."""
    Q, K, V = _inputs(7, 2, 4, 2, 70, 90, 64, torch.bfloat16, cuda)
    att = rkv.SinkAttention(device=cuda)
    lens = torch.tensor([90, 33], dtype=torch.int32, device=cuda)
    want = torch.zeros_like(Q)
    att(Q, K, V, lens=lens, out=want)
    assert torch.equal(att(Q, K, V, lens=lens), want) and bool((want[1, :, 13:] == 0).all())
    att(Q, K, V, out=want)

    def fill(*args, **kw):
        raise AssertionError("an output was filled")

    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", fill)
        got = att(Q, K, V)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Lq,Lk", [(600, 600), (40, 6000)])
def test_a_non_finite_key_stays_in_the_queries_that_see_it(dtype, D, bad, Lq, Lk, cuda):
    """Queries before it and those whose window has passed it keep their bits,
    though their tiles hold it, and so do other KV heads' queries."""
    H, HK, window = 4, 2, 17
    Q, K, V = _inputs(8, 1, H, HK, Lq, Lk, D, dtype, cuda)
    j = Lk - Lq + 20
    ref, got = (torch.zeros_like(Q) for _ in range(2))
    lse0, lse = (torch.zeros((1, H, Lq), device=cuda) for _ in range(2))
    att = rkv.SinkAttention(sinks=3, window=window, device=cuda)
    att(Q, K, V, out=ref, lse=lse0)
    K[0, 1, j, 2] = bad
    att(Q, K, V, out=got, lse=lse)
    p = torch.arange(Lk - Lq, Lk, device=cuda)
    sees = torch.zeros((1, H, Lq), dtype=torch.bool, device=cuda)
    sees[0, H // HK:] = (p >= j) & (p < j + window)
    assert torch.equal(got[~sees], ref[~sees]) and torch.equal(lse[~sees], lse0[~sees])
    if math.isnan(bad):
        assert bool(got[sees].isnan().all())
