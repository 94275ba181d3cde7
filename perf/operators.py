"""The operators over a paged KV cache, and the sink-window prefill attention
that fills it, as a user's program runs them: one token attended over a paged
cache, new rows appended to the pages, eviction by accumulated attention
weight, and causal attention over a sliding window with a few first tokens
that stay visible.

``own`` false computes each operator in plain torch operations in 32 bits;
``own`` true calls the library.  Sizes are the repository's own geometries
(24 query and 8 KV heads of 128, 2048- to 131072-token caches, the 3717-token
cache that budget 1024 leaves of an 8192-token prompt) and generic ones.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _package():
    here = os.path.join(os.getcwd(), "rocketkv-cpp_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import rocketkv_b200
    return rocketkv_b200


# ---- the cases ---------------------------------------------------------------

def _decode(name, batch, heads, kv_heads, dim, dtype, page, length, ragged=False, sinks=0, window=0, weights=False, mix=0):
    return dict(name=name, op="decode", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page,
                length=length, ragged=ragged, sinks=sinks, window=window, weights=weights, mix=mix)


def _append(name, batch, kv_heads, dim, dtype, page, length, rows, ragged=False, mix=0):
    return dict(name=name, op="append", batch=batch, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, length=length,
                rows=rows, ragged=ragged, mix=mix)


def _evict(name, batch, kv_heads, dim, dtype, page, length, budget, sinks, recent, ragged=False, mix=0):
    return dict(name=name, op="evict", batch=batch, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, length=length,
                budget=budget, sinks=sinks, recent=recent, ragged=ragged, mix=mix)


def _prefill(name, batch, heads, kv_heads, dim, dtype, queries, keys, sinks, window, ragged=False, mix=0):
    return dict(name=name, op="prefill", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                queries=queries, keys=keys, sinks=sinks, window=window, ragged=ragged, mix=mix)


def listed():
    return [
        # one layer's step of a single user over a 2048-token cache: latency
        _decode("decode 1x2048", 1, 24, 8, 128, "bf16", 16, 2048),
        # one layer's step of a full serving batch, prompts of every length up to 8192
        _decode("decode 64 ragged 8192", 64, 24, 8, 128, "bf16", 16, 8192, ragged=True, mix=1),
        # long contexts that nothing was evicted from
        _decode("decode 8x131072", 8, 24, 8, 128, "bf16", 64, 131072),
        # a step that also accumulates each token's attention weight, on the cache budget 1024 leaves of an 8192-token prompt
        _decode("decode weights 16x3717", 16, 24, 8, 128, "f16", 32, 3717, weights=True),
        # fp32, no shared heads, an odd page size and length, a window with sinks
        _decode("decode window f32", 5, 8, 8, 64, "f32", 24, 4099, ragged=True, sinks=4, window=1024, mix=2),
        # the new token's row of every sequence of a batch
        _append("append 64x1", 64, 8, 128, "bf16", 16, 8192, 1, ragged=True, mix=1),
        # prompts of several lengths put into pages
        _append("append 6x2048", 6, 8, 128, "f16", 32, 2048, 2048, ragged=True, mix=3),
        # one sequence that has grown 64 tokens over its budget
        _evict("evict 1x2112", 1, 8, 128, "bf16", 16, 2112, 2048, 4, 32),
        # a batch cut to budget 1024, some of it shorter than that
        _evict("evict 64 ragged 3717", 64, 8, 128, "bf16", 16, 3717, 1024, 4, 32, ragged=True, mix=4),
        # long contexts cut to budget 4096
        _evict("evict 8x131072", 8, 8, 128, "f16", 64, 131072, 4096, 4, 256),
        # the prefill of an 8192-token prompt over a window of 2048 and 4 sinks
        _prefill("prefill 8192 window 2048", 1, 24, 8, 128, "bf16", 8192, 8192, 4, 2048),
        # a padded batch of short prompts behind a cached prefix, another head size
        _prefill("prefill 3 ragged 1537", 3, 8, 2, 64, "f16", 1289, 1537, 4, 250, ragged=True, mix=5),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "append", "evict", "prefill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, 96, 256])
    mix = rng.randrange(1 << 20)
    ragged = rng.random() < 0.6
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "prefill":
        heads, kv_heads = rng.choice([(24, 8), (8, 8), (8, 2), (8, 1)])
        keys = _log(rng, 64, min(8000, int((7e10 / (heads * dim)) ** 0.5)))
        queries = keys if rng.random() < 0.5 else rng.randint(1, keys)
        batch = rng.randint(1, max(1, min(6, int(7e10 / (heads * dim * queries * keys)))))
        window = 0 if rng.random() < 0.25 else _log(rng, 1, keys)
        return {k: v for k, v in _prefill("", batch, heads, kv_heads, dim, dtype, queries, keys, rng.choice([0, 1, 4, 40]), window,
                                          ragged, mix).items() if k != "name"}
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    length = _log(rng, 16, 131072)
    row = kv_heads * dim * SIZE[dtype] * 2
    batch = _log(rng, 1, max(1, min(64, int(1.2e9 / (row * length)))))
    if op == "decode":
        window = _log(rng, 1, length) if rng.random() < 0.4 else 0
        d = _decode("", batch, kv_heads * rng.choice([1, 3, 4, 8, 12]), kv_heads, dim, dtype, page, length, ragged, rng.choice([0, 4, 33]),
                    window, rng.random() < 0.4, mix)
    elif op == "append":
        d = _append("", batch, kv_heads, dim, dtype, page, length, 1 if rng.random() < 0.4 else _log(rng, 1, length), ragged, mix)
    else:
        sinks, recent = min(length - 1, rng.choice([0, 4])), _log(rng, 1, max(1, length // 4))
        low = sinks + recent
        d = _evict("", batch, kv_heads, dim, dtype, page, length, rng.randint(min(low, length), length), sinks, min(recent, max(0, length - sinks)),
                   ragged, mix)
        d["budget"] = max(d["budget"], d["sinks"] + d["recent"])
    return {k: v for k, v in d.items() if k != "name"}


def _lengths(case, top):
    """Tokens of each sequence: all `top`, or spread over 0 .. top with the first at `top`."""
    if not case["ragged"]:
        return [top] * case["batch"]
    r = random.Random(case["mix"])
    return [top] + [r.randint(0, top) for _ in range(case["batch"] - 1)]


def _rows(case):
    """New rows of each sequence of an append."""
    lengths = _lengths(case, case["length"])
    if not case["ragged"]:
        return [min(case["rows"], n) for n in lengths]
    r = random.Random(case["mix"] + 1)
    return [min(n, case["rows"] if i == 0 or case["rows"] == 1 else r.randint(0, case["rows"])) for i, n in enumerate(lengths)]


# ---- inputs --------------------------------------------------------------------

def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _pool(case, g, tokens_each, dtype, fill=True):
    """K and V pages [pages][KV heads][page][dim] and a table of every sequence's pages, in a mixed order."""
    per = -(-max(tokens_each, 1) // case["page"])
    pages = case["batch"] * per + 3
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    table = torch.randperm(pages, generator=g, device="cuda")[: case["batch"] * per].view(case["batch"], per).to(torch.int32)
    if not fill:
        return torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda"), table
    K, V = torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda")
    for at in range(0, pages, 4096):
        K[at: at + 4096] = _randn(g, K[at: at + 4096].shape, dtype)
        V[at: at + 4096] = _randn(g, V[at: at + 4096].shape, dtype)
    # one key in a hundred stands out, as salient tokens do
    stand = torch.rand(shape[:3], generator=g, device="cuda") < 0.01
    K.mul_(torch.where(stand, 4.0, 1.0).to(dtype)[..., None])
    return K, V, table


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, s = TYPES[case["dtype"]], {"case": case}
    rkv = _package() if own else None
    if case["op"] == "prefill":
        B, H, HK, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        s["Q"], s["K"], s["V"] = (_randn(g, (B, n, t, D), dtype) for n, t in ((H, case["queries"]), (HK, case["keys"]), (HK, case["keys"])))
        s["lens"] = _ints(_lengths(case, case["keys"])) if case["ragged"] else None
        s["O"] = torch.zeros_like(s["Q"])
        s["lse"] = torch.zeros((B, H, case["queries"]), dtype=torch.float32, device="cuda")
        if own:
            s["attention"] = rkv.SinkAttention(sinks=case["sinks"], window=case["window"], device="cuda")
        return s
    s["K"], s["V"], s["table"] = _pool(case, g, case["length"], dtype)
    s["lens"] = _ints(_lengths(case, case["length"]))
    if own:
        s["cache"] = rkv.PagedCache(s["K"], s["V"], s["table"], s["lens"])
    B, HK, D = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "decode":
        s["Q"] = _randn(g, (B, case["heads"], D), dtype)
        s["weights"] = torch.rand((B, HK, case["length"]), generator=g, device="cuda") if case["weights"] else None
        if own:
            s["decoder"] = rkv.PagedDecoder(case["heads"], HK, D, case["length"], B, "cuda", sinks=case["sinks"], window=case["window"],
                                            weights=case["weights"])
    elif case["op"] == "append":
        s["n_new"] = _ints(_rows(case))
        # K and V rows as a fused projection leaves them: one buffer, token-major
        s["kv"] = _randn(g, (B, case["rows"], 2 * HK, D), dtype)
        s["k"], s["v"] = s["kv"][:, :, :HK], s["kv"][:, :, HK:]
    else:
        w = torch.randn((B, HK, case["length"]), generator=g, device="cuda").exp_()
        # weights repeat among rarely attended tokens: every second one in steps of 1/8
        coarse = (w * 8).round_() / 8
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.5, coarse, w)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["K_out"], s["V_out"], s["table_out"] = _pool(case, g, min(case["budget"], case["length"]), dtype, fill=False)
        if own:
            s["out"] = rkv.PagedCache(s["K_out"], s["V_out"], s["table_out"], None)
            s["evictor"] = rkv.WeightEvictor(HK, case["length"], B, case["budget"], "cuda", sinks=case["sinks"], recent=case["recent"])
    return s


# ---- the operators ---------------------------------------------------------------

def run(state):
    return {"decode": _run_decode, "append": _run_append, "evict": _run_evict, "prefill": _run_prefill}[state["case"]["op"]](state)


def _gather(pool, table, t):
    """Rows [batch][KV heads][tokens][dim] of the tokens t [tokens] of every sequence."""
    page = pool.shape[2]
    return pool[table[:, t // page].long(), :, (t % page)[None].expand(table.shape[0], -1)].transpose(1, 2)


def _softmax(logits, seen):
    """Weights and log-sum-exp over the last axis; a row that sees nothing gets zeros and -inf."""
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0), (torch.log(total) + top).squeeze(-1)


def _run_decode(s):
    c = s["case"]
    if own:
        s["decoder"](s["Q"], s["cache"], s["weights"])
        return {"O": s["decoder"].O, "lse": s["decoder"].lse} | ({"weights": s["weights"]} if c["weights"] else {})
    B, H, HK, D, L = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["length"]
    t = torch.arange(L, device="cuda")
    lens = s["lens"][:, None]
    seen = t < lens
    if c["window"]:
        seen &= (t < c["sinks"]) | (t >= lens - c["window"])
    q = s["Q"].float().view(B, HK, H // HK, D)
    logits = torch.matmul(q, _gather(s["K"], s["table"], t).float().transpose(2, 3)) / math.sqrt(D)
    p, lse = _softmax(logits, seen[:, None, None])
    V = _gather(s["V"], s["table"], t).float().masked_fill(~seen[:, None, :, None], 0.0)
    out = {"O": torch.matmul(p, V).view(B, H, D), "lse": lse.reshape(B, H)}
    if c["weights"]:
        s["weights"] += p.sum(2)
        out["weights"] = s["weights"]
    return out


def _run_append(s):
    c = s["case"]
    if own:
        _package().paged_append(s["cache"], s["k"], s["v"], s["n_new"])
        return {"K": s["K"], "V": s["V"]}
    n = s["n_new"][:, None].long()
    t = torch.arange(c["rows"], device="cuda")[None].minimum((n - 1).clamp(min=0))  # past the last row: that row again
    slot = (s["lens"][:, None].long() - n + t).clamp(0, c["length"] - 1)
    pages, at = s["table"].long().gather(1, slot // c["page"]), slot % c["page"]
    item = torch.arange(c["batch"], device="cuda")[:, None]
    for pool, rows in ((s["K"], s["k"]), (s["V"], s["v"])):
        pool[pages, :, at] = torch.where((n > 0)[..., None, None], rows[item, t], pool[pages, :, at])
    return {"K": s["K"], "V": s["V"]}


def _run_evict(s):
    c = s["case"]
    if own:
        kept, new_lens = s["evictor"](s["cache"], s["weights"], out=s["out"], weights_out=s["weights_out"])
        return {"kept": kept, "new_lens": new_lens, "weights": s["weights_out"], "K": s["K_out"], "V": s["V_out"]}
    L, m = c["length"], min(c["budget"], c["length"])
    t = torch.arange(L, device="cuda")
    lens = s["lens"][:, None, None]
    rank = s["weights"].masked_fill((t < c["sinks"]) | (t >= lens - c["recent"]), math.inf).masked_fill(t >= lens, -math.inf)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :m]
    new = lens.clamp(max=c["budget"])
    i = torch.arange(m, device="cuda")
    kept = best.masked_fill(i >= new, L).sort(dim=-1).values
    have = kept < L
    src = kept.clamp(max=L - 1)
    w = torch.zeros_like(s["weights"])
    w[..., :m] = s["weights"].gather(-1, src).masked_fill(~have, 0.0)
    item, head = torch.arange(c["batch"], device="cuda")[:, None, None], torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    pages, at = s["table"].long()[item, src // c["page"]], src % c["page"]
    to, place = s["table_out"].long()[item, i // c["page"]], (i % c["page"])[None, None]
    for pool, out in ((s["K"], s["K_out"]), (s["V"], s["V_out"])):
        out[to, head, place] = torch.where(have[..., None], pool[pages, head, at], out[to, head, place])
    return {"kept": kept.masked_fill(~have, -1).to(torch.int32), "new_lens": new.reshape(-1).to(torch.int32), "weights": w, "K": s["K_out"],
            "V": s["V_out"]}


def _run_prefill(s):
    c = s["case"]
    if own:
        s["attention"](s["Q"], s["K"], s["V"], lens=s["lens"], out=s["O"], lse=s["lse"])
        return {"O": s["O"], "lse": s["lse"]}
    B, H, HK, D, Lq, Lk = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["queries"], c["keys"]
    p = torch.arange(Lq, device="cuda")[:, None] + (Lk - Lq)
    j = torch.arange(Lk, device="cuda")
    seen = j <= p
    if c["window"]:
        seen &= (j < c["sinks"]) | (j > p - c["window"])
    q = s["Q"].float().view(B, HK, H // HK, Lq, D)
    logits = torch.matmul(q, s["K"].float().transpose(2, 3)[:, :, None]).mul_(1 / math.sqrt(D))
    w, lse = _softmax(logits, seen)
    O = torch.matmul(w, s["V"].float()[:, :, None]).view(B, H, Lq, D).to(s["Q"].dtype)
    lse = lse.reshape(B, H, Lq)
    if s["lens"] is not None:  # rows of queries behind a sequence's end stay as they were
        real = p.view(-1) < s["lens"][:, None, None]
        O, lse = torch.where(real[..., None], O, s["O"]), torch.where(real, lse, s["lse"])
    return {"O": O, "lse": lse}


# ---- what a pass cannot do without ---------------------------------------------------

def _visible(case, n):
    return min(n, case["sinks"] + case["window"]) if case["window"] else n


def work(case):
    D, size = case["dim"], SIZE[case["dtype"]]
    if case["op"] == "prefill":
        B, H, HK = case["batch"], case["heads"], case["kv_heads"]
        off = case["keys"] - case["queries"]
        pairs = rows = read = 0
        for n in _lengths(case, case["keys"]):
            if n > off:
                rows += n - off
                pairs += sum(_visible(case, p + 1) for p in range(off, n))
                first = max(0, off - case["window"] + 1) if case["window"] else 0
                read += n if first <= case["sinks"] else n - first + case["sinks"]
        return {"bytes": size * D * (2 * H * rows + 2 * HK * read) + 4 * H * rows, "flops": 4 * H * D * pairs}
    HK, lengths = case["kv_heads"], _lengths(case, case["length"])
    if case["op"] == "decode":
        seen = sum(_visible(case, n) for n in lengths)
        return {"bytes": seen * HK * (2 * D * size + (8 if case["weights"] else 0)) + case["batch"] * case["heads"] * (D * (size + 4) + 4),
                "flops": 4 * case["heads"] * D * seen}
    if case["op"] == "append":
        rows = sum(_rows(case))
        return {"bytes": 4 * rows * HK * D * size, "flops": 0}
    new = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": HK * (4 * sum(lengths) + 4 * case["batch"] * case["length"] + 4 * new + 4 * new * D * size), "flops": HK * sum(lengths)}


# ---- the operators in 64 bits, from their definitions ----------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return None  # rows are copied, nothing is computed
    if case["op"] == "decode":
        B, H, HK, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        G = H // HK
        O = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
        lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
        W = s["weights"].double() if case["weights"] else None
        for b, n in enumerate(_lengths(case, case["length"])):
            at = [t for t in range(n) if not case["window"] or t < case["sinks"] or t >= n - case["window"]] if case["window"] else None
            t = torch.arange(n, device="cuda") if at is None else torch.tensor(at, device="cuda", dtype=torch.int64)
            if t.numel() == 0:
                continue
            pages = s["table"][b].long()[t // case["page"]]
            for h in range(HK):
                k, v = (x[pages, h, t % case["page"]].double() for x in (s["K"], s["V"]))
                l = s["Q"][b, h * G:(h + 1) * G].double() @ k.T / D ** 0.5
                lse[b, h * G:(h + 1) * G] = torch.logsumexp(l, 1)
                p = torch.softmax(l, 1)
                O[b, h * G:(h + 1) * G] = p @ v
                if W is not None:
                    W[b, h, t] += p.sum(0)
        return {"O": O, "lse": lse} | ({"weights": W} if case["weights"] else {})
    if case["op"] == "evict":
        m, sinks, recent = min(case["budget"], case["length"]), case["sinks"], case["recent"]
        w, W, kept = s["weights"].double().cpu(), torch.zeros(s["weights"].shape, dtype=torch.float64), []
        for b, n in enumerate(_lengths(case, case["length"])):
            for h in range(case["kv_heads"]):
                keep = list(range(n))
                if n > case["budget"]:
                    x = w[b, h].tolist()
                    middle = sorted(range(sinks, n - recent), key=lambda t: (-x[t], t))[: case["budget"] - sinks - recent]
                    keep = list(range(sinks)) + sorted(middle) + list(range(n - recent, n))
                W[b, h, : len(keep)] = w[b, h, torch.tensor(keep, dtype=torch.int64)]
                kept.append(keep + [-1] * (m - len(keep)))
        new = [min(n, case["budget"]) for n in _lengths(case, case["length"])]
        return {"kept": torch.tensor(kept).view(case["batch"], case["kv_heads"], m), "new_lens": torch.tensor(new), "weights": W, "K": None, "V": None}
    B, H, HK, Lq, Lk = case["batch"], case["heads"], case["kv_heads"], case["queries"], case["keys"]
    O = torch.zeros(s["Q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, H, Lq), dtype=torch.float64, device="cuda")
    p, j = torch.arange(Lk - Lq, Lk, device="cuda")[:, None], torch.arange(Lk, device="cuda")[None]
    hidden = j > p
    if case["window"]:
        hidden |= (j >= case["sinks"]) & (j <= p - case["window"])
    for b, n in enumerate(_lengths(case, Lk)):
        rows = max(0, n - (Lk - Lq))
        for h in range(H if rows else 0):
            l = s["Q"][b, h, :rows].double() @ s["K"][b, h // (H // HK)].double().T / case["dim"] ** 0.5
            l.masked_fill_(hidden[:rows], -math.inf)
            lse[b, h, :rows] = torch.logsumexp(l, 1)
            O[b, h, :rows] = torch.softmax(l, 1) @ s["V"][b, h // (H // HK)].double()
    return {"O": O, "lse": lse}
