"""Rotary positions on the GPU, alone and on the way into the paged cache,
against the formula in 64 bits."""
import math

import pytest
import torch

import pagedref as R
import rocketkv_b200 as rkv

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _freqs(pairs, base=500000.0):
    return base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)


def _axes(pairs, n):
    return None if n == 1 else torch.arange(pairs) * n // pairs


def _turn(x, positions, freqs, axes, interleaved):
    """Rows x [B, heads, n, D] turned, and how far the kernel may be off.  The
    angle: an fp32 of half turns below 1 (2^-25 of one), cut to 32 bits
    (2^-31), the frequency and its product's wrap (2^-33 at 2^31); the sine and
    cosine of it are good to 2 ulp (2^-23 at 1); two products and their sum in
    fp32 (three halves of 2^-23 of the terms); one rounding to the type, whose
    smallest step counts for fp16."""
    pairs = len(freqs)
    y = x.double().clone()
    lo = y[..., 0: 2 * pairs: 2] if interleaved else y[..., :pairs]
    hi = y[..., 1: 2 * pairs: 2] if interleaved else y[..., pairs: 2 * pairs]
    ax = torch.zeros(pairs, dtype=torch.long) if axes is None else axes
    t = (positions.double()[ax.to(x.device)] * freqs.to(x.device)[:, None, None]).permute(1, 2, 0)[:, None]  # [B, 1, n, pairs]
    a, b = lo.clone(), hi.clone()
    lo.copy_(a * t.cos() - b * t.sin())
    hi.copy_(a * t.sin() + b * t.cos())
    tol = torch.zeros_like(y)
    each = (a.abs() + b.abs()) * (math.pi * (2.0 ** -25 + 2.0 ** -30) + 2.0 ** -23 + 1.5 * 2.0 ** -23)
    (tol[..., 0: 2 * pairs: 2] if interleaved else tol[..., :pairs]).copy_(each)
    (tol[..., 1: 2 * pairs: 2] if interleaved else tol[..., pairs: 2 * pairs]).copy_(each)
    if x.dtype != torch.float32:
        tol[..., : 2 * pairs] += R.unit(x.dtype) * (y.abs() + tol)[..., : 2 * pairs]
        if x.dtype == torch.float16:
            tol[..., : 2 * pairs] += 2.0 ** -25
    return y, tol


def _positions(seed, axes, B, n, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    p = torch.randint(0, 1 << 20, (axes, B, n), generator=g, device=dev)
    p[..., 0] = 0
    if n > 2:
        p[..., 1] = -(1 << 31)
        p[..., 2] = (1 << 31) - 1
    return p.to(torch.int32)


# (type, D, H, HK, pairs, axes, interleaved, B, len)
ROTATE = [
    ("bf16", 128, 24, 8, 64, 1, False, 1, 513),
    ("bf16", 128, 24, 8, 64, 3, False, 3, 67),
    ("f16", 128, 4, 1, 64, 2, True, 2, 33),
    ("f32", 96, 8, 2, 24, 1, True, 3, 37),
    ("f32", 64, 3, 3, 32, 4, False, 2, 5),
    ("bf16", 80, 5, 5, 20, 1, False, 2, 9),     # 8-byte vectors
    ("f16", 72, 2, 1, 9, 3, False, 2, 11),      # single elements
    ("bf16", 72, 2, 1, 13, 1, True, 1, 7),
    ("f32", 8, 1, 1, 1, 1, True, 1, 1),
    ("f32", 256, 2, 1, 127, 1, False, 1, 3),
    ("bf16", 256, 16, 2, 128, 3, True, 1, 4097),
    ("f16", 16, 1, 0, 8, 1, False, 65, 2),
]


@pytest.mark.parametrize("case", ROTATE, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("layout", ["fused", "heads", "in place", "odd"])
def test_rotate_against_64_bits(case, layout, cuda):
    kind, D, H, HK, pairs, na, inter, B, n = case
    dt = TYPES[kind]
    g = torch.Generator(device=cuda).manual_seed(5)
    fr, ax = _freqs(pairs), _axes(pairs, na)
    pos = _positions(6, na, B, n, cuda)
    flat = torch.randn(B * n * (H + HK) * D + 1, generator=g, device=cuda).to(dt)
    if layout in ("heads", "in place"):
        q, k = flat[: B * H * n * D].view(B, H, n, D), flat[B * H * n * D: -1].view(B, HK, n, D)
    else:
        fused = flat[int(layout == "odd"):][: B * n * (H + HK) * D].view(B, n, H + HK, D)
        q, k = fused[:, :, :H].transpose(1, 2), fused[:, :, H:].transpose(1, 2)
    if HK == 0:
        k = None
    want = [None if x is None else _turn(x, pos, fr, ax, inter) for x in (q, k)]
    before = flat.clone()
    r = rkv.Rotary(fr, D, axes=ax, num_axes=na, interleaved=inter, device=cuda)
    outs = (q, k) if layout == "in place" else (torch.full((B, n, H, D), 7.0, dtype=dt, device=cuda).transpose(1, 2), None)
    got = rkv.rotate(q, k, pos, r, q_out=outs[0], k_out=outs[1])
    for x, w in zip(got, want):
        if w is not None:
            y, tol = w
            assert bool(((x.double() - y).abs() <= tol).all()), float(((x.double() - y).abs() / tol.clamp(min=1e-30)).max())
            assert torch.equal(x[..., 2 * pairs:].double(), y[..., 2 * pairs:])
    if layout != "in place":
        assert torch.equal(flat, before)


def test_rotation_by_the_negative_position_is_its_gradient(cuda):
    """The rotation is linear and orthogonal: <turn(x), g> = <x, turn'(g)>, and
    a difference along any direction gives the same."""
    B, H, n, D = 2, 3, 50, 64
    g = torch.Generator(device=cuda).manual_seed(1)
    x, up, step = (torch.randn((B, H, n, D), generator=g, device=cuda) for _ in range(3))
    pos = _positions(2, 1, B, n, cuda).clamp(min=-(1 << 31) + 1)
    r = rkv.Rotary(_freqs(32), D, device=cuda)
    back = rkv.rotate(up, None, -pos, r)[0]
    along = rkv.rotate(x + step, None, pos, r)[0].double() - rkv.rotate(x, None, pos, r)[0].double()
    # each of the 2 sums' terms is good to about 2^-21 of it
    scale = float((along.abs() * up.abs().double()).sum())
    assert abs(float((along * up).sum() - (back.double() * step).sum())) <= 2.0 ** -20 * scale


def test_pairs_of_an_axis_without_positions_are_copied(cuda):
    x = torch.randn((1, 2, 4, 16), device=cuda)
    pos = _positions(3, 1, 1, 4, cuda)
    r = rkv.Rotary(_freqs(8), 16, axes=[0] * 8, device=cuda)
    r.axes[4:] = 1
    got = rkv.rotate(x, None, pos, r)[0]
    assert torch.equal(got[..., 4:8], x[..., 4:8]) and torch.equal(got[..., 12:], x[..., 12:])
    assert not torch.equal(got[..., :4], x[..., :4])


def test_rotate_keeps_non_finite_values_in_their_pairs(cuda):
    x = torch.randn((1, 1, 3, 32), device=cuda)
    x[0, 0, 1, 3] = math.nan
    x[0, 0, 2, 20] = math.inf
    got = rkv.rotate(x, None, torch.arange(3, dtype=torch.int32, device=cuda)[None] + 5, rkv.Rotary(_freqs(16), 32, device=cuda))[0]
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[0, 0, 1, [3, 19]] = True
    want[0, 0, 2, [4, 20]] = True
    assert torch.equal(bad, want)


# (type, D, H, HK, page, layout, pairs, axes, interleaved, given)
APPEND = [
    ("bf16", 128, 24, 8, 16, "hnd", 64, 1, False, False),
    ("bf16", 128, 24, 8, 16, "nhd", 64, 3, False, True),
    ("f16", 64, 4, 2, 24, "mixed", 32, 2, True, True),
    ("f32", 8, 3, 3, 1, "hnd", 2, 1, True, False),
    ("bf16", 72, 5, 5, 7, "hnd", 13, 1, False, False),
    ("f32", 256, 0, 2, 64, "hnd", 64, 1, False, True),
]


def _cache(seed, B, hk, d, page, top, dtype, dev, layout, lens):
    per = max(1, -(-top // page))
    K, V = R.pool(seed, B * per + 3, hk, page, d, dtype, dev, layout)
    return rkv.PagedCache(K, V, R.table(seed + 1, B, per, B * per + 3, dev), torch.tensor(lens, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("T", [37, 1])
def test_append_rotated_against_64_bits(case, odd, T, cuda):
    """Ragged counts, rows of a fused buffer; every other row of the pages and
    of q_out stays as it was."""
    kind, D, H, HK, page, layout, pairs, na, inter, given = case
    dt, B, top = TYPES[kind], 5, 100
    lens, n_new = [100, 40, 1, 0, 64], [min(T, x) for x in (37, 0, 1, 0, 20)]
    c = _cache(70, B, HK, D, page, top, dt, cuda, layout, lens)
    K0, V0 = c.K.double(), c.V.clone()
    width = H + 2 * HK
    flat = torch.randn(B * T * width * D + 1, device=cuda).to(dt)
    q, k, v = flat[int(odd): int(odd) + B * T * width * D].view(B, T, width, D).split([H, HK, HK], dim=2)
    fr, ax = _freqs(pairs), _axes(pairs, na)
    pos = _positions(7, na, B, T, cuda)
    full = pos if given else torch.stack([torch.arange(T, device=cuda) + (a - b) for a, b in zip(lens, n_new)]).expand(na, -1, -1)
    kw, kt = _turn(k.transpose(1, 2), full, fr, ax, inter)
    qw, qt = _turn(q.transpose(1, 2), full, fr, ax, inter)
    r = rkv.Rotary(fr, D, axes=ax, num_axes=na, interleaved=inter, device=cuda)
    q_out = torch.full((B, T, H, D), 7.0, dtype=dt, device=cuda)
    got = rkv.paged_append_rotated(c, k, v, r, q=q if H else None, q_out=q_out if H else None, positions=pos if given else None,
                                   n_new=torch.tensor(n_new, dtype=torch.int32, device=cuda))
    tolK = torch.zeros_like(K0)
    for b in range(B):
        for i in range(n_new[b]):
            t = lens[b] - n_new[b] + i
            p, row = int(c.block_table[b, t // page]), t % page
            K0[p, :, row], tolK[p, :, row], V0[p, :, row] = kw[b, :, i], kt[b, :, i], v[b, i]
    assert bool(((c.K.double() - K0).abs() <= tolK).all()) and torch.equal(c.V, V0)
    if not H:
        assert got is None
        return
    assert got.data_ptr() == q_out.data_ptr()
    for b in range(B):
        n = n_new[b]
        assert bool(((q_out[b, :n].transpose(0, 1).double() - qw[b, :, :n]).abs() <= qt[b, :, :n]).all())
        assert bool((q_out[b, n:] == 7.0).all())


def test_append_rotated_equals_rotate_then_append(cuda):
    """Bit for bit, and one step's [B, heads, D] form."""
    B, H, HK, D, page = 3, 6, 2, 64, 16
    c = _cache(80, B, HK, D, page, 60, torch.bfloat16, cuda, "hnd", [60, 33, 7])
    d = rkv.PagedCache(c.K.clone(), c.V.clone(), c.block_table, c.lens)
    q, k, v = (torch.randn((B, n, D), device=cuda).to(torch.bfloat16) for n in (H, HK, HK))
    pos = torch.tensor([1000, 5, 0], dtype=torch.int32, device=cuda)
    r = rkv.Rotary(_freqs(32), D, device=cuda)
    got = rkv.paged_append_rotated(c, k, v, r, q=q, positions=pos)
    qr, kr = rkv.rotate(q[:, :, None], k[:, :, None], pos[:, None].contiguous(), r)
    rkv.paged_append(d, kr[:, :, 0], v)
    assert got.shape == (B, H, D) and torch.equal(got, qr[:, :, 0])
    assert torch.equal(c.K, d.K) and torch.equal(c.V, d.V)


def test_append_rotated_skips_what_has_no_place(cuda):
    """Rows behind the table or on pages outside the pool are left out of the
    pages; their queries are turned all the same.  Counts are clamped."""
    B, H, HK, D, page = 4, 2, 2, 64, 16
    c = _cache(75, B, HK, D, page, 32, torch.float32, cuda, "hnd", [2, 40, 32, 20])
    c.block_table[2, 1] = -7
    k, v = (torch.randn((B, 10, HK, D), device=cuda) for _ in range(2))
    q = torch.randn((B, 10, H, D), device=cuda)
    n_new = torch.tensor([10, 10, 99, -3], dtype=torch.int32, device=cuda)
    fr = _freqs(32)
    K0, V0, tolK = c.K.double(), c.V.clone(), torch.zeros(c.K.shape, dtype=torch.float64, device=cuda)
    first = torch.tensor([2 - 10, 40 - 10, 32 - 10, 20], device=cuda)
    pos = (first[:, None] + torch.arange(10, device=cuda))[None]
    kw, kt = _turn(k.transpose(1, 2), pos, fr, None, False)
    qw, qt = _turn(q.transpose(1, 2), pos, fr, None, False)
    q_out = torch.full_like(q, 7.0)
    rkv.paged_append_rotated(c, k, v, rkv.Rotary(fr, D, device=cuda), q=q, q_out=q_out, n_new=n_new)
    for b, (n, m) in enumerate(((2, 10), (40, 10), (32, 10), (20, 0))):
        for i in range(m):
            t = n - m + i
            if 0 <= t < 32 and 0 <= int(c.block_table[b, t // page]) < c.K.shape[0]:
                p = int(c.block_table[b, t // page])
                K0[p, :, t % page], tolK[p, :, t % page], V0[p, :, t % page] = kw[b, :, i], kt[b, :, i], v[b, i]
        assert bool(((q_out[b, :m].transpose(0, 1).double() - qw[b, :, :m]).abs() <= qt[b, :, :m]).all())
        assert bool((q_out[b, m:] == 7.0).all())
    assert bool(((c.K.double() - K0).abs() <= tolK).all()) and torch.equal(c.V, V0)


def test_rotary_calls_on_another_stream_and_in_a_graph(cuda):
    B, H, HK, n, D = 2, 6, 2, 130, 128
    q, k = (torch.randn((B, h, n, D), device=cuda).to(torch.bfloat16) for h in (H, HK))
    pos = _positions(9, 1, B, n, cuda)
    r = rkv.Rotary(_freqs(64), D, device=cuda)
    want = rkv.rotate(q, k, pos, r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = rkv.rotate(q, k, pos, r, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c = _cache(90, B, HK, D, 16, 200, torch.bfloat16, cuda, "hnd", [200, 140])
    rows = [x.transpose(1, 2) for x in (k, k, q)]
    q_out = torch.zeros((B, n, H, D), dtype=torch.bfloat16, device=cuda)
    rkv.paged_append_rotated(c, rows[0], rows[1], r, q=rows[2], q_out=q_out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rkv.paged_append_rotated(c, rows[0], rows[1], r, q=rows[2], q_out=q_out)
    for lens in ([130, 131], [200, 199]):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.normal_()
        k.normal_()
        K = c.K.clone()
        g.replay()
        d = rkv.PagedCache(K, c.V.clone(), c.block_table, c.lens)
        wq = rkv.paged_append_rotated(d, rows[0], rows[1], r, q=rows[2])
        assert torch.equal(q_out, wq) and torch.equal(c.K, K) and torch.equal(c.V, d.V)


def test_empty_calls(cuda):
    r = rkv.Rotary(_freqs(8), 16, device=cuda)
    e = torch.empty((0, 2, 3, 16), device=cuda)
    assert rkv.rotate(e, None, torch.empty((0, 3), dtype=torch.int32, device=cuda), r)[0].shape == e.shape
    e = torch.empty((2, 2, 0, 16), device=cuda)
    assert rkv.rotate(e, e, torch.empty((2, 0), dtype=torch.int32, device=cuda), r)[1].shape == e.shape


def test_refused_calls(cuda):
    r = rkv.Rotary(_freqs(8), 16, device=cuda)
    x = torch.randn((2, 2, 3, 16), device=cuda)
    pos = torch.zeros((2, 3), dtype=torch.int32, device=cuda)
    for bad in (dict(q=x, k=x.bfloat16()), dict(q=x, k=x[:1]), dict(q=x[0], k=None), dict(q=x, k=None, positions=pos[:1]),
                dict(q=x, k=None, positions=pos.float()), dict(q=x, k=None, q_out=x[:, :1]), dict(q=x, k=None, q_out=x.bfloat16()),
                dict(q=x[..., :8], k=None), dict(q=x.transpose(2, 3), k=None), dict(q=x, k=None, positions=pos.t().contiguous())):
        with pytest.raises((ValueError, TypeError)):
            rkv.rotate(**{**dict(positions=pos, rotary=r), **bad})
    with pytest.raises(rkv.RkvError):  # rows that are written would meet
        rkv.rotate(x, None, pos, r, q_out=torch.empty((2, 1, 3, 16), device=cuda).expand(2, 2, 3, 16))
