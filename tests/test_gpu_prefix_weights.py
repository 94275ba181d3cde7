"""Weights of the shared tokens in the shared-prefix decode: they keep 16 bits
or more, whichever kernel attends them, as the decode of every sequence alone
does.  Neighbouring tokens have nearly the same weight and opposite values, so
that what is left of the output is the weights' difference."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv
from test_gpu_prefix import _query, _setup

pytestmark = pytest.mark.gpu


def _opposite(cache, tokens, page, dtype):
    """Values of odd tokens are those of the token before, negated; keys
    those of the token before but for one column."""
    at = cache.block_table[0].long()
    for t in range(1, tokens, 2):
        a, b = (at[(t - 1) // page], (t - 1) % page), (at[t // page], t % page)
        cache.V[b[0], :, b[1]] = -cache.V[a[0], :, a[1]]
        k = cache.K[a[0], :, a[1]].clone()
        k[:, 0] = (k[:, 0].float() * 0.5 + 1.0).to(dtype)
        cache.K[b[0], :, b[1]] = k


@pytest.mark.parametrize("kind,D,H,B", [("bf16", 128, 12, 50), ("f16", 128, 12, 50), ("bf16", 64, 4, 30), ("f16", 256, 12, 30),
                                        ("bf16", 256, 4, 40), ("bf16", 128, 12, 2), ("f16", 128, 12, 2)])
@pytest.mark.parametrize("tokens", [32, 64, 200])
def test_weights_of_shared_tokens_keep_16_bits(kind, D, H, B, tokens, cuda):
    """Bounds: a score's (a dot product of D terms, the rounding of the
    exponent's argument) and the sums' in fp32, as in the decode's other tests;
    a weight in two 16-bit parts is off by the square of half a step of the type
    (the second part is rounded, the first one's rest is exact), in fp16 by 2^-32
    of the row's largest at least; the output's rounding."""
    dt = {"bf16": torch.bfloat16, "f16": torch.float16}[kind]
    HK, page = 2, 8
    cache, starts, shared = _setup(400 + tokens, HK, D, page, [(tokens, [tokens] * B)], dt, cuda)
    _opposite(cache, tokens, page, dt)
    Q = (_query(401, B, H, D, dt, cuda).float() * 0.125).to(dt)
    dec = rkv.PrefixDecoder(H, HK, D, tokens, B, dt, cuda)
    dec(Q, cache, starts, shared)
    t = torch.arange(tokens)
    k, v = (R.rows(P, cache.block_table, 0, t).double().transpose(0, 1)[None] for P in (cache.K, cache.V))
    q = Q.double().view(B, HK, H // HK, D)
    s = q @ k.transpose(2, 3) / math.sqrt(D)
    mag = q.abs() @ k.abs().transpose(2, 3) / math.sqrt(D)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    p = e / total
    O = p @ v
    es = R.EPS * (R.LAM * math.sqrt(D + 2) * mag + 4 * s.abs() + 4 * m.abs() + 8)
    sums = R.EPS * (R.LAM * math.sqrt(tokens) + 8)
    u = R.unit(dt)
    pv = p @ v.abs()
    tol = (p * (es + u * u)) @ v.abs() + ((p * es).sum(-1, keepdim=True) + 2 * sums) * pv + u * O.abs()
    if kind == "f16":
        tol = tol + 2.0 ** -32 * v.abs().sum(2, keepdim=True) / total + 2.0 ** -25
    off = (dec.O.view_as(O).double() - O).abs()
    assert float(O.abs().max()) > 50 * float(tol.median())  # there is something left to be right
    assert bool((off <= tol).all()), float((off / tol).max())
