"""Rotary positions, the paged append that applies them on the way, and the
decode of a batch whose sequences share long prefixes, as a user's program
runs them next to the paged cache and the sink-window prefill.

``own`` false computes each operator in plain torch operations in 32 bits
(angles in 64); ``own`` true calls the library.  Sizes are the repository's own
geometries (24 query and 8 KV heads of 128, 2048- to 131072-token caches) and
generic ones.
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

def _rotate(name, batch, heads, kv_heads, dim, dtype, tokens, pairs, axes=1, interleaved=False, mix=0):
    return dict(name=name, op="rotate", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, tokens=tokens, pairs=pairs,
                axes=axes, interleaved=interleaved, mix=mix)


def _append(name, batch, heads, kv_heads, dim, dtype, page, length, rows, pairs, axes=1, interleaved=False, given=True, ragged=False, mix=0):
    return dict(name=name, op="append", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, length=length,
                rows=rows, pairs=pairs, axes=axes, interleaved=interleaved, given=given, ragged=ragged, mix=mix)


def _prefix(name, batch, heads, kv_heads, dim, dtype, page, prefix, own_tokens, groups=1, ragged=False, mix=0):
    return dict(name=name, op="prefix", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, prefix=prefix,
                own_tokens=own_tokens, groups=groups, ragged=ragged, mix=mix)


def listed():
    return [
        # the query and key rows of one user's short prompt: latency
        _rotate("rotate 1x512", 1, 24, 8, 128, "bf16", 512, 64),
        # prompts with images, positions in time, height and width
        _rotate("rotate 3 axes 4x4096", 4, 24, 8, 128, "bf16", 4096, 64, axes=3, mix=1),
        # fp32, neighbouring columns as pairs, half of the columns rotated, an odd length
        _rotate("rotate interleaved f32 3x1537", 3, 8, 2, 96, "f32", 1537, 24, interleaved=True, mix=2),
        # the new token of every sequence of a batch, its position kept apart from the cache's length (as after evictions)
        _append("append 64x1", 64, 24, 8, 128, "bf16", 16, 2048, 1, 64, ragged=True, mix=3),
        # prompts with images put into pages
        _append("append 3 axes 6x2048", 6, 24, 8, 128, "f16", 32, 2048, 2048, 64, axes=3, ragged=True, mix=4),
        # a piece of each prompt behind what the cache holds, positions by the cache's length
        _append("append f32 5x333", 5, 8, 8, 64, "f32", 24, 1500, 333, 16, interleaved=True, given=False, ragged=True, mix=5),
        # two answers to one short prompt: latency
        _prefix("prefix 2x1024+64", 2, 24, 8, 128, "bf16", 16, 1024, 64),
        # a full serving batch behind one system prompt, a slot of it idle
        _prefix("prefix 64x8192+512", 64, 24, 8, 128, "bf16", 16, 8192, 512, ragged=True, mix=6),
        # questions on one very long document
        _prefix("prefix 8x131072+1024", 8, 24, 8, 128, "bf16", 64, 131072, 1024, ragged=True, mix=7),
        # many samples of four prompts
        _prefix("prefix 4 groups 192x4096+256", 192, 16, 2, 128, "f16", 32, 4096, 256, groups=4, ragged=True, mix=8),
        # fp32, no shared heads, an odd page size
        _prefix("prefix f32 6x4080+300", 6, 8, 8, 64, "f32", 24, 4080, 300, ragged=True, mix=9),
        # heads of 256
        _prefix("prefix 256 wide 24x4096+128", 24, 16, 2, 256, "bf16", 16, 4096, 128, mix=10),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 128, 128, 96, 80, 256])
    mix = rng.randrange(1 << 20)
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    heads, kv_heads = rng.choice([(24, 8), (24, 8), (8, 8), (8, 2), (16, 2), (8, 1), (12, 4)])
    if op == "prefix":
        own_tokens = rng.choice([0, 1, _log(rng, 2, 2048), _log(rng, 2, 2048)])
        row = kv_heads * dim * SIZE[dtype] * 2
        prefix = max(page, _log(rng, 64, min(131072, int(5e8 / row))) // page * page)
        groups = max(1, min(rng.randint(1, 6) if rng.random() < 0.4 else 1, int(3e8 / (row * prefix))))
        most = min(256, 2e8 / (row * (own_tokens + 1)), 3e10 / (heads * dim * (prefix + own_tokens)) / (2 if dtype == "f32" else 1))
        batch = max(groups, _log(rng, 1, max(1, int(most))))
        d = _prefix("", batch, heads, kv_heads, dim, dtype, page, prefix, own_tokens, groups, rng.random() < 0.7, mix)
        return {k: v for k, v in d.items() if k != "name"}
    pairs = rng.choice([dim // 2, dim // 2, dim // 4, rng.randint(1, dim // 2)])
    axes = rng.choice([1, 1, 2, 3])
    interleaved = rng.random() < 0.3
    row = (heads + kv_heads) * dim * SIZE[dtype]
    tokens = _log(rng, 1, min(16384, int(1.3e8 / row)))
    batch = _log(rng, 1, max(1, min(64, int(1.3e8 / (row * tokens)))))
    if op == "rotate":
        d = _rotate("", batch, heads, kv_heads, dim, dtype, tokens, pairs, axes, interleaved, mix)
    else:
        rows = 1 if rng.random() < 0.4 else tokens
        d = _append("", batch, heads, kv_heads, dim, dtype, page, max(tokens, rng.randint(1, 2048)), rows, pairs, axes, interleaved,
                    rng.random() < 0.6, rng.random() < 0.6, mix)
    return {k: v for k, v in d.items() if k != "name"}


def _lengths(case):
    """Tokens of each sequence of an append, the new ones counted, and how many those are."""
    B, top, rows = case["batch"], case["length"], min(case["rows"], case["length"])
    if not case["ragged"]:
        return [top] * B, [rows] * B
    r = random.Random(case["mix"])
    lens = [top] + [r.randint(0, top) for _ in range(B - 1)]
    return lens, [min(n, rows if i == 0 or rows == 1 else r.randint(0, rows)) for i, n in enumerate(lens)]


def _groups(case):
    """First sequence of each group (and the batch behind them), the groups' shared tokens (whole pages), every sequence's own tokens;
    a ragged batch of 8 or more ends with an idle slot, which has no tokens at all."""
    B, n, page = case["batch"], case["groups"], case["page"]
    r = random.Random(case["mix"])
    starts = [B * g // n for g in range(n + 1)]
    shared = [max(page, case["prefix"] // page * page)] * n
    tokens = [case["own_tokens"]] * B
    if case["ragged"]:
        starts[1:n] = sorted(r.sample(range(1, B), n - 1)) if n > 1 else []
        shared[1:] = [r.randint(max(1, shared[0] // page // 4), shared[0] // page) * page for _ in range(n - 1)]
        tokens[1:] = [r.randint(0, case["own_tokens"]) for _ in range(B - 1)]
    idle = case["ragged"] and B >= 8
    of = [max(g for g in range(n) if starts[g] <= b) for b in range(B)]
    lens = [0 if idle and b == B - 1 else shared[of[b]] + tokens[b] for b in range(B)]
    return starts, shared, of, lens


# ---- inputs --------------------------------------------------------------------

def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(g, shape, dtype):
    P = torch.empty(shape, dtype=dtype, device="cuda")
    for at in range(0, shape[0], 4096):
        P[at: at + 4096] = _randn(g, P[at: at + 4096].shape, dtype)
    return P


def _frequencies(case):
    """Radians per position of each pair, and the axis that it turns with: a quarter of the pairs with the first, the rest shared by the others."""
    pairs, axes = case["pairs"], case["axes"]
    i = torch.arange(pairs)
    axis = ((i - pairs // 4) * (axes - 1) // (pairs - pairs // 4) + 1).masked_fill(i < pairs // 4, 0) if axes > 1 else torch.zeros_like(i)
    return 500000.0 ** (-i.double() / pairs), axis


def _positions(case, g, rows):
    """[axes, batch, rows]: the first counts on from some far position, the others go over grids."""
    t = torch.arange(rows, device="cuda")
    first = torch.randint(0, 1 << 20, (case["batch"], 1), generator=g, device="cuda")
    width = torch.randint(3, 60, (case["batch"], 1), generator=g, device="cuda")
    return torch.stack([first + t, first + t // width, first + t % width][: case["axes"]]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, s = TYPES[case["dtype"]], {"case": case}
    rkv = _package() if own else None
    B, H, HK, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "prefix":
        starts, shared, of, lens = _groups(case)
        page, per = case["page"], max(1, -(-max(lens) // case["page"]), max(shared) // case["page"])
        own_pages = [-(-max(0, n - shared[of[b]]) // page) for b, n in enumerate(lens)]
        total = sum(shared) // page + sum(own_pages) + 3
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        table, at, group_pages = [], 0, []
        for p in shared:
            group_pages.append(order[at: at + p // page])
            at += p // page
        for b in range(B):
            mine = group_pages[of[b]] + order[at: at + own_pages[b]]
            at += own_pages[b]
            table.append(mine + [0] * (per - len(mine)))
        s["K"], s["V"] = (_pool(g, (total, HK, page, D), dtype) for _ in range(2))
        # one key in a hundred stands out, as salient tokens do
        s["K"].mul_(torch.where(torch.rand(s["K"].shape[:3], generator=g, device="cuda") < 0.01, 4.0, 1.0).to(dtype)[..., None])
        s["table"], s["lens"], s["starts"], s["shared"] = _ints(table), _ints(lens), _ints(starts), _ints(shared)
        s["Q"] = _randn(g, (B, H, D), dtype)
        if own:
            s["cache"] = rkv.PagedCache(s["K"], s["V"], s["table"], s["lens"])
            s["decoder"] = rkv.PrefixDecoder(H, HK, D, max(lens), B, dtype, "cuda", num_groups=case["groups"])
        return s
    s["inv_freq"], s["axes"] = (x.cuda() for x in _frequencies(case))
    if own:
        f, a = _frequencies(case)
        s["rotary"] = rkv.Rotary(f, D, axes=a, interleaved=case["interleaved"], device="cuda")
    # Q, K and V rows as a fused projection leaves them: one buffer, token-major
    rows = case["tokens"] if case["op"] == "rotate" else min(case["rows"], case["length"])
    s["qkv"] = _randn(g, (B, rows, H + 2 * HK, D), dtype)
    s["q"], s["k"], s["v"] = s["qkv"].split([H, HK, HK], dim=2)
    s["positions"] = _positions(case, g, rows)
    if case["op"] == "rotate":
        s["q"], s["k"] = s["q"].transpose(1, 2), s["k"].transpose(1, 2)
        s["q_out"], s["k_out"] = (torch.zeros((B, n, rows, D), dtype=dtype, device="cuda") for n in (H, HK))
        return s
    lens, n_new = _lengths(case)
    per = max(1, -(-case["length"] // case["page"]))
    pages = B * per + 3
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[: B * per].view(B, per).to(torch.int32)
    s["K"], s["V"] = (_pool(g, (pages, HK, case["page"], D), dtype) for _ in range(2))
    s["lens"], s["n_new"] = _ints(lens), _ints(n_new)
    s["q_out"] = torch.zeros((B, rows, H, D), dtype=dtype, device="cuda")
    if own:
        s["cache"] = rkv.PagedCache(s["K"], s["V"], s["table"], s["lens"])
    return s


# ---- the operators ---------------------------------------------------------------

def run(state):
    return {"rotate": _run_rotate, "append": _run_append, "prefix": _run_prefix}[state["case"]["op"]](state)


def _turned(x, positions, s):
    """Rows x [..., D] with their pairs turned; positions [axes, ...] broadcast against x without its columns."""
    c = s["case"]
    pairs = c["pairs"]
    angle = positions[s["axes"]].movedim(0, -1).double() * s["inv_freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    y = x.float()
    turn, rest = y[..., : 2 * pairs], y[..., 2 * pairs:]
    if c["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        both = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turn[..., :pairs], turn[..., pairs:]
        both = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([both, rest], -1).to(x.dtype)


def _run_rotate(s):
    if own:
        _package().rotate(s["q"], s["k"], s["positions"], s["rotary"], q_out=s["q_out"], k_out=s["k_out"])
        return {"q": s["q_out"], "k": s["k_out"]}
    return {"q": _turned(s["q"], s["positions"][:, :, None], s), "k": _turned(s["k"], s["positions"][:, :, None], s)}


def _run_append(s):
    c = s["case"]
    if own:
        _package().paged_append_rotated(s["cache"], s["k"], s["v"], s["rotary"], q=s["q"], q_out=s["q_out"],
                                        positions=s["positions"] if c["given"] else None, n_new=s["n_new"])
        return {"K": s["K"], "V": s["V"], "q": s["q_out"]}
    rows = s["qkv"].shape[1]
    n = s["n_new"][:, None].long()
    i = torch.arange(rows, device="cuda")[None]
    token = s["lens"][:, None].long() - n + i
    positions = s["positions"] if c["given"] else token.expand(c["axes"], -1, -1)
    q, k = _turned(s["q"], positions[..., None], s), _turned(s["k"], positions[..., None], s)
    last = i.minimum((n - 1).clamp(min=0))  # past the last row: that row again
    slot = (token - i + last).clamp(0, c["length"] - 1)
    pages, at = s["table"].long().gather(1, slot // c["page"]), slot % c["page"]
    item = torch.arange(c["batch"], device="cuda")[:, None]
    for pool, x in ((s["K"], k), (s["V"], s["v"])):
        pool[pages, :, at] = torch.where((n > 0)[..., None, None], x[item, last], pool[pages, :, at])
    return {"K": s["K"], "V": s["V"], "q": torch.where((i < n)[..., None, None], q, s["q_out"])}


def _gather(pool, table, t):
    """Rows [sequences][KV heads][tokens][dim] of the tokens t [sequences or 1][tokens] of a table's sequences."""
    page = pool.shape[2]
    t = t.expand(table.shape[0], -1)
    return pool[table.long().gather(1, t // page), :, t % page].transpose(1, 2).float()


def _run_prefix(s):
    c = s["case"]
    if own:
        s["decoder"](s["Q"], s["cache"], s["starts"], s["shared"])
        return {"O": s["decoder"].O, "lse": s["decoder"].lse}
    B, H, HK, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    G, Gr, P, N = H // HK, c["groups"], s["table"].shape[1] * c["page"], max(1, c["own_tokens"])
    P = min(P, max(c["page"], c["prefix"] // c["page"] * c["page"]))
    b = torch.arange(B, device="cuda")
    of = torch.bucketize(b, s["starts"][1:].long(), right=True)  # the sequence's group, and its place there
    place = b - s["starts"][of]
    size = B  # of a group at most
    lens, shared = s["lens"].long(), s["shared"].long()
    if Gr > 1:
        size = B - Gr + 1 if c["ragged"] else -(-B // Gr)
    q = torch.zeros((Gr, size, HK, G, D), device="cuda")
    q[of, place] = s["Q"].float().view(B, HK, G, D)
    # the shared tokens: every group's rows at once against its first sequence's pages
    t = torch.arange(P, device="cuda")[None]
    first = s["table"][s["starts"][:-1].long()]
    x = torch.matmul(q.transpose(1, 2).reshape(Gr, HK, size * G, D), _gather(s["K"], first, t).transpose(2, 3))
    x = x.view(Gr, HK, size, G, P).transpose(1, 2)[of, place]
    x = x.masked_fill_(~((t < shared[of][:, None]) & (lens > 0)[:, None])[:, None, None], -math.inf)
    # each sequence's own
    at = shared[of][:, None] + torch.arange(N, device="cuda")
    mine = at < lens[:, None]
    at = at.clamp(max=s["table"].shape[1] * c["page"] - 1)
    y = torch.matmul(s["Q"].float().view(B, HK, G, D), _gather(s["K"], s["table"], at).transpose(2, 3))
    x = torch.cat([x, y.masked_fill(~mine[:, None, None], -math.inf)], -1).div_(math.sqrt(D))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    lse = (total.log() + top).reshape(B, H)
    x = x.div_(torch.where(total > 0, total, 1.0))
    w = torch.zeros((Gr, size, HK, G, P), device="cuda")
    w[of, place] = x[..., :P]
    O = torch.matmul(w.transpose(1, 2).reshape(Gr, HK, size * G, P), _gather(s["V"], first, t))
    O = O.view(Gr, HK, size, G, D).transpose(1, 2)[of, place]
    O = O + torch.matmul(x[..., P:], _gather(s["V"], s["table"], at).masked_fill(~mine[:, None, :, None], 0.0))
    return {"O": O.reshape(B, H, D).to(s["Q"].dtype), "lse": lse}


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    B, H, HK, D, size = case["batch"], case["heads"], case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    if case["op"] == "rotate":
        rows = B * case["tokens"]
        return {"bytes": rows * (2 * (H + HK) * D * size + 4 * case["axes"]), "flops": 6 * rows * (H + HK) * case["pairs"]}
    if case["op"] == "append":
        rows = sum(_lengths(case)[1])
        return {"bytes": rows * (2 * (H + 2 * HK) * D * size + 4 * case["axes"] * case["given"]), "flops": 6 * rows * (H + HK) * case["pairs"]}
    _, shared, of, lens = _groups(case)
    once = sum(shared) + sum(max(0, n - shared[of[b]]) for b, n in enumerate(lens))
    return {"bytes": 2 * HK * D * size * once + B * H * (2 * D * size + 4), "flops": 4 * H * D * sum(lens)}


# ---- the operators in 64 bits, from their definitions ----------------------------------

def _exact_rows(x, positions, case):
    """Rows [batch, tokens, heads, D] turned, as complex numbers; positions [axes, batch, tokens]."""
    f, axes = _frequencies(case)
    n = case["pairs"]
    y = x.double().clone()
    lo = y[..., 0: 2 * n: 2] if case["interleaved"] else y[..., :n]
    hi = y[..., 1: 2 * n: 2] if case["interleaved"] else y[..., n: 2 * n]
    angle = torch.stack([positions[int(a)].double() * float(w) for w, a in zip(f, axes)], -1)
    z = torch.complex(lo.contiguous(), hi.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
    lo.copy_(z.real)
    hi.copy_(z.imag)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    B, H, HK, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        return {x: _exact_rows(s[x].transpose(1, 2), s["positions"], case).transpose(1, 2) for x in ("q", "k")}
    if case["op"] == "append":
        lens, n_new = _lengths(case)
        rows = s["qkv"].shape[1]
        if not case["given"]:
            s["positions"] = torch.stack([torch.arange(rows, device="cuda") + (n - m) for n, m in zip(lens, n_new)]).expand(case["axes"], -1, -1)
        q, k = _exact_rows(s["q"], s["positions"], case), _exact_rows(s["k"], s["positions"], case)
        K, Q = s["K"].double(), s["q_out"].double()
        for b, (n, m) in enumerate(zip(lens, n_new)):
            t = torch.arange(n - m, n, device="cuda")
            K[s["table"][b].long()[t // case["page"]], :, t % case["page"]] = k[b, :m]
            Q[b, :m] = q[b, :m]
        return {"K": K, "V": None, "q": Q}
    G = H // HK
    O = torch.zeros((B, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_groups(case)[3]):
        t = torch.arange(n, device="cuda")
        pages = s["table"][b].long()[t // case["page"]]
        for h in range(HK if n else 0):
            k, v = (x[pages, h, t % case["page"]].double() for x in (s["K"], s["V"]))
            l = s["Q"][b, h * G:(h + 1) * G].double() @ k.T / D ** 0.5
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(l, 1)
            O[b, h * G:(h + 1) * G] = torch.softmax(l, 1) @ v
    return {"O": O, "lse": lse}
