"""Plain 64-bit forms of the paged-cache operators and of the sink-window
attention, and the error bounds the tests hold the kernels to."""
import math

import torch

EPS = 2.0 ** -24  # half a step of fp32, relative
LAM = 6.0         # a sum of n rounded terms is off by LAM sqrt(n) EPS times the terms' magnitude


def unit(dtype):
    """Half a step of a type, relative."""
    return torch.finfo(dtype).eps / 2


def pool(seed, pages, hk, page, d, dtype, device, layout="hnd", scale=1.0):
    """K and V pages [pages, HK, page, D] in one of three memory layouts."""
    g = torch.Generator(device=device).manual_seed(seed)
    shape = {"hnd": (2, pages, hk, page, d), "nhd": (2, pages, page, hk, d), "mixed": (pages, 2, page, hk, d)}[layout]
    buf = (torch.randn(shape, generator=g, device=device) * scale).to(dtype)
    if layout == "hnd":
        return buf[0], buf[1]
    if layout == "nhd":
        return buf[0].transpose(1, 2), buf[1].transpose(1, 2)
    return buf[:, 0].transpose(1, 2), buf[:, 1].transpose(1, 2)


def table(seed, batch, per, pages, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[: batch * per].view(batch, per).to(torch.int32).to(device)


def rows(P, tab, b, tokens):
    """Rows [tokens, HK, D] of sequence b."""
    page = P.shape[2]
    t = torch.as_tensor(tokens, dtype=torch.int64, device=P.device)
    return P[tab[b].long()[t // page], :, t % page]


def seen(n, sinks, window):
    t = torch.arange(n)
    return t if not window else t[(t < sinks) | (t >= n - window)]


def decode(Q, K, V, tab, lens, sinks=0, window=0, skip=()):
    """O, lse, per-token weights (list of [HK, n]) and bounds on the fp32 error
    of each: the scores' (a dot product of D terms, then the rounding of the
    exponent's argument), carried through the softmax, and the sums'."""
    B, H, D = Q.shape
    HK = K.shape[1]
    G = H // HK
    dev = Q.device
    O = torch.zeros((B, H, D), dtype=torch.float64, device=dev)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=dev)
    tolO, tolL = torch.zeros_like(O), torch.zeros_like(lse)
    W, tolW = [], []
    for b in range(B):
        n = int(lens[b])
        w, tw = (torch.zeros((HK, n), dtype=torch.float64, device=dev) for _ in range(2))
        t = torch.tensor([int(x) for x in seen(n, sinks, window) if (b, int(x)) not in skip], dtype=torch.int64, device=dev)
        for h in range(HK if len(t) else 0):
            q = Q[b, h * G:(h + 1) * G].double()
            k, v = rows(K, tab, b, t)[:, h].double(), rows(V, tab, b, t)[:, h].double()
            s = q @ k.T / math.sqrt(D)
            mag = q.abs() @ k.abs().T / math.sqrt(D)
            m = s.amax(1, keepdim=True)
            e = torch.exp(s - m)
            p = e / e.sum(1, keepdim=True)
            O[b, h * G:(h + 1) * G] = p @ v
            lse[b, h * G:(h + 1) * G] = (m + e.sum(1, keepdim=True).log()).squeeze(1)
            # relative error of each exponential
            es = EPS * (LAM * math.sqrt(D + 2) * mag + 4 * s.abs() + 4 * m.abs() + 8)
            cap = es.amax(1, keepdim=True)
            sums = EPS * (LAM * math.sqrt(len(t)) + 8)
            rel = (p * es).sum(1, keepdim=True) + sums  # of the sum of exponentials
            tolO[b, h * G:(h + 1) * G] = (p * es) @ v.abs() + (rel + sums) * (p @ v.abs())
            tolL[b, h * G:(h + 1) * G] = (cap + sums + EPS * (4 + lse[b, h * G:(h + 1) * G, None].abs())).squeeze(1)
            w[h, t] = p.sum(0)
            # fp32 has no normal numbers below 2^-126 (its last step is 2^-149), and an exponential down there may
            # be flushed to zero: each of the G terms of a weight is off by up to 2^-126 whatever its size
            tw[h, t] = (p * (es + rel)).sum(0) + 4 * EPS * p.sum(0) + G * 2.0 ** -126
        W.append(w)
        tolW.append(tw)
    return O, lse, W, tolO + 1e-37, tolL, tolW


def kept_lists(weights, lens, budget, sinks, recent):
    """Kept token lists [B][HK] of python ints."""
    out = []
    for b in range(len(lens)):
        n = int(lens[b])
        per = []
        for h in range(weights.shape[1]):
            if n <= budget:
                per.append(list(range(n)))
                continue
            w = weights[b, h, :n].double().cpu().tolist()
            rank = lambda t: (0, -w[t], t) if w[t] == w[t] else (1, 0.0, t)  # noqa: E731
            mid = sorted(range(sinks, n - recent), key=rank)[: budget - sinks - recent]
            per.append(list(range(sinks)) + sorted(mid) + list(range(n - recent, n)))
        out.append(per)
    return out


def sink_attention(Q, K, V, sinks, window, lens=None):
    """O, lse and the error bounds; rows at positions from lens on are NaN."""
    B, H, Lq, D = Q.shape
    HK, Lk = K.shape[1], K.shape[2]
    G = H // HK
    dev = Q.device
    uT = unit(Q.dtype)
    O = torch.full(Q.shape, math.nan, dtype=torch.float64, device=dev)
    lse = torch.full((B, H, Lq), math.nan, dtype=torch.float64, device=dev)
    tolO, tolL = torch.zeros_like(O), torch.zeros_like(lse)
    j = torch.arange(Lk, device=dev)[None]
    for b in range(B):
        n = Lk if lens is None else int(lens[b])
        r = max(0, n - (Lk - Lq))
        p_ = torch.arange(Lk - Lq, Lk - Lq + r, device=dev)[:, None]
        see = (j <= p_) & (j < n)
        if window:
            see &= (j < sinks) | (j > p_ - window)
        for h in range(H if r else 0):
            q, k, v = Q[b, h, :r].double(), K[b, h // G, :n].double(), V[b, h // G, :n].double()
            s = (q @ k.T / math.sqrt(D)).masked_fill(~see[:, :n], -math.inf)
            mag = (q.abs() @ k.abs().T / math.sqrt(D)).masked_fill(~see[:, :n], 0.0)
            m = s.amax(1, keepdim=True)
            e = torch.exp(s - m)
            p = e / e.sum(1, keepdim=True)
            O[b, h, :r] = p @ v
            lse[b, h, :r] = (m + e.sum(1, keepdim=True).log()).squeeze(1)
            sf = s.masked_fill(s == -math.inf, 0.0).abs()
            # an exponential is rounded to Q's type before it meets V where that has 16 bits
            es = EPS * (LAM * math.sqrt(D + 2) * mag + 4 * sf + 4 * m.abs() + 8)
            ep = es + (uT if Q.dtype != torch.float32 else 0.0)
            sums = EPS * (LAM * math.sqrt(n) + 8)
            rel = (p * es).sum(1, keepdim=True) + sums
            pv = p @ v.abs()
            tolO[b, h, :r] = (p * ep) @ v.abs() + (rel + sums) * pv + uT * (O[b, h, :r].abs() + uT * pv)
            # fp16 weights below 2^-14 of the row's largest have a fixed step of 2^-24
            if Q.dtype == torch.float16:
                tolO[b, h, :r] += 2.0 ** -25 * (see[:, :n].double() @ v.abs()) / e.sum(1, keepdim=True)
                tolO[b, h, :r] += 2.0 ** -25  # an output below 2^-14
            tolL[b, h, :r] = ((es * see[:, :n]).amax(1, keepdim=True) + sums + EPS * (4 + lse[b, h, :r, None].abs())).squeeze(1)
    return O, lse, tolO + 1e-37, tolL
