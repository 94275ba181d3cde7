"""Eviction by accumulated weight on long caches: every variant of the
selection (keys in shared memory or not, one CTA or a cluster per list), with
the last weight that stays a NaN, an infinity, a zero of either sign, a negative number
or one of many equal, in sequences far shorter than the bound on their length
too."""
import math

import numpy as np
import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu

# the weights that the competing tokens fall back to, once fewer than the budget have an ordinary one
FILL = {
    "nan": lambda r, n: np.full(n, math.nan),
    "-inf": lambda r, n: np.full(n, -math.inf),
    "nan and -inf": lambda r, n: np.where(r.random(n) < 0.5, math.nan, -math.inf),
    "inf": lambda r, n: np.full(n, math.inf),
    "zeros": lambda r, n: np.where(r.random(n) < 0.5, 0.0, -0.0),
    "one negative": lambda r, n: np.full(n, -1.5),
    "negative": lambda r, n: -np.exp(r.standard_normal(n)),
    "tiny": lambda r, n: np.where(r.random(n) < 0.5, 1e-45, -1e-45),
}


def _weights(seed, lens, heads, top, budget, fill):
    r = np.random.default_rng(seed)
    w = np.full((len(lens), heads, top), 1e30, dtype=np.float32)  # behind the end: must not be ranked
    for b, n in enumerate(lens):
        for h in range(heads):
            w[b, h, :n] = FILL[fill](r, n)
            some = r.permutation(n)[: budget * 9 // 10]
            w[b, h, some] = np.exp(r.standard_normal(len(some)))
    return w


def _kept(w, lens, budget, sinks, recent):
    """[B, HK, min(budget, top)] by a stable sort: NaN last, larger first, lower index first."""
    B, heads, top = w.shape
    out = np.full((B, heads, min(budget, top)), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        for h in range(heads):
            keep = np.arange(n)
            if n > budget:
                x = w[b, h, sinks: n - recent].astype(np.float64)
                nan = np.isnan(x)
                order = np.lexsort((-np.where(nan, 0.0, x) + 0.0, nan))[: budget - sinks - recent]
                keep = np.concatenate((np.arange(sinks), np.sort(order) + sinks, np.arange(n - recent, n)))
            out[b, h, : len(keep)] = keep
    return out


# batch, KV heads, max_len, budget, sinks, recent, lens in turn
SHAPES = {
    "shared memory, one CTA": (20, 4, 9001, 1000, 4, 32, [2000, 9001, 1001, 5000, 1000, 0]),
    "shared memory, cluster": (2, 2, 20000, 3000, 0, 1, [20000, 3001]),
    "one CTA": (10, 8, 40960, 1000, 4, 32, [2000, 17000, 40960, 1001, 999, 33000, 12345, 1, 0, 24000]),
    "one CTA, odd rows": (19, 4, 33003, 700, 0, 0, [800, 2000, 16000, 33003, 701]),
    "cluster": (1, 2, 300000, 5000, 10, 100, [300000]),
    "cluster, short": (2, 2, 280001, 2000, 4, 0, [9000, 30000]),
}


@pytest.mark.parametrize("fill", list(FILL))
@pytest.mark.parametrize("shape", list(SHAPES))
def test_thresholds_on_odd_weights(shape, fill, cuda):
    B, HK, top, budget, sinks, recent, lens = SHAPES[shape]
    lens = [lens[b % len(lens)] for b in range(B)]
    page, D = 64, 8
    per, per_out = -(-top // page), -(-budget // page)
    K, V = R.pool(1, B * per, HK, page, D, torch.bfloat16, cuda)
    Ko, Vo = R.pool(2, B * per_out, HK, page, D, torch.bfloat16, cuda)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    c = rkv.PagedCache(K, V, R.table(3, B, per, B * per, cuda), n)
    out = rkv.PagedCache(Ko, Vo, R.table(4, B, per_out, B * per_out, cuda), None)
    w = _weights(5, lens, HK, top, budget, fill)
    want = torch.from_numpy(_kept(w, lens, budget, sinks, recent)).to(cuda)
    W = torch.from_numpy(w).to(cuda)
    Wo = torch.full_like(W, -3.0)
    ev = rkv.WeightEvictor(HK, top, B, budget, cuda, sinks=sinks, recent=recent)

    here, at = want >= 0, want.clamp(min=0)
    item, head = torch.arange(B, device=cuda)[:, None, None], torch.arange(HK, device=cuda)[None, :, None]
    rows = [P[c.block_table.long()[item, at // page], head, at % page].clone() for P in (K, V)]
    We = torch.zeros_like(W)
    We[:, :, : want.shape[2]] = W.gather(2, at).masked_fill(~here, 0.0)

    def check(kept, new, weights, cache):
        assert torch.equal(kept.long(), want)
        assert new.tolist() == [min(x, budget) for x in lens]
        assert torch.equal(weights.isnan(), We.isnan()) and torch.equal(weights.nan_to_num(7.0), We.nan_to_num(7.0))
        i = torch.arange(want.shape[2], device=cuda)
        page_of, slot = cache.block_table.long()[:, i // page][:, None], (i % page)[None, None]
        for P, x in zip((cache.K, cache.V), rows):
            assert torch.equal(P[page_of, head, slot][here], x[here])

    check(*ev(c, W, out=out, weights_out=Wo), Wo, out)
    check(*ev(c, W), W, c)
