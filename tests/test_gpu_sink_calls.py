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
