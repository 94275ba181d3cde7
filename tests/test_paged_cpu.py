"""Refusals of the paged-cache and sink-attention entry points, and their size
queries: host logic only, nothing is launched."""
import ctypes

import pytest

import rocketkv_b200 as rkv

INV, UNS, WS, OK = rkv.RKV_ERR_INVALID_ARG, rkv.RKV_ERR_UNSUPPORTED, rkv.RKV_ERR_WORKSPACE, rkv.RKV_OK
P = 1 << 20  # stands for a device address: never followed


def cache(**kw):
    f = dict(K=P, V=P, dtype=rkv.BF16, num_heads_kv=2, dim_head=64, page_size=16, num_pages=4, table_stride=2,
             page_stride=2 * 16 * 128, head_stride=16 * 128, token_stride=128, block_table=P, lens=P)
    f.update(kw)
    return rkv._PagedCache(**f)


BAD_CACHES = [
    (dict(dtype=rkv.Q8_0), INV), (dict(dtype=9), INV), (dict(num_heads_kv=0), INV), (dict(page_size=0), INV),
    (dict(num_pages=-1), INV), (dict(table_stride=-1), INV), (dict(dim_head=0), INV), (dict(dim_head=60), UNS),
    (dict(dim_head=264), UNS), (dict(K=P + 8), INV), (dict(V=P + 2), INV), (dict(token_stride=120), INV),
    (dict(token_stride=136), INV), (dict(head_stride=64), INV), (dict(page_stride=0), INV), (dict(K=None), INV),
    (dict(V=None), INV), (dict(block_table=None), INV), (dict(lens=None), INV),
]


def append(c, k=P, v=P, n=1, batch=1, item=256, tok=256, head=128, n_new=None):
    return rkv.lib().rkv_paged_append(ctypes.byref(c) if c else None, k, v, n, batch, item, tok, head, n_new, None)


def decode(c, Q=P, qs=4 * 128, H=4, max_len=32, batch=1, sinks=0, window=0, O=P, lse=None, w=None, wst=0, ws=P, wb=1 << 30):
    return rkv.lib().rkv_paged_decode(Q, qs, H, ctypes.byref(c) if c else None, max_len, batch, sinks, window, O, lse, w,
                                      wst, ws, wb, None)


def evict(c, w=P, wst=32, max_len=32, batch=1, budget=16, sinks=2, recent=2, out=None, wo=None, kept=P, kst=16, new=P + 64):
    return rkv.lib().rkv_weight_evict(ctypes.byref(c) if c else None, w, wst, max_len, batch, budget, sinks, recent,
                                      ctypes.byref(out) if out else None, wo, kept, kst, new, None)


@pytest.mark.parametrize("kw,want", BAD_CACHES, ids=lambda x: str(x))
def test_bad_caches_are_refused(kw, want):
    c = cache(**kw)
    assert append(c) == want and decode(c) == want and evict(c) == want


def test_no_cache():
    assert append(None) == INV and decode(None) == INV and evict(None) == INV


def test_append_arguments():
    c = cache()
    assert append(c, k=None) == INV and append(c, v=None) == INV
    assert append(c, n=-1) == INV and append(c, batch=-1) == INV
    assert append(c, k=P + 1) == INV and append(c, n=2, tok=129) == INV and append(c, head=-2) == INV
    assert append(c, batch=70000) == UNS
    assert append(c, n=0) == OK and append(c, batch=0) == OK  # nothing to do


def test_decode_arguments():
    c = cache()
    assert decode(c, H=3) == INV and decode(c, H=0) == INV and decode(c, Q=None) == INV and decode(c, O=None) == INV
    assert decode(c, Q=P + 8) == INV and decode(c, batch=2, qs=8) == INV and decode(c, batch=2, qs=4 * 128 + 8) == INV
    assert decode(c, sinks=-1) == INV and decode(c, window=-1) == INV and decode(c, max_len=-1) == INV
    assert decode(c, max_len=(1 << 30) + 1) == UNS
    assert decode(c, w=P, wst=31) == INV
    assert decode(c, ws=None) == WS and decode(c, ws=P + 4) == WS and decode(c, wb=8) == WS
    assert decode(c, batch=0) == OK


def test_evict_arguments():
    c = cache()
    assert evict(c, w=None) == INV and evict(c, wst=31) == INV and evict(c, kept=None) == INV and evict(c, kst=15) == INV
    assert evict(c, new=None) == INV and evict(c, new=P) == INV  # lens cannot be overwritten while it is read
    assert evict(c, budget=-1) == INV and evict(c, sinks=15, recent=2) == INV and evict(c, recent=-1) == INV
    assert evict(c, max_len=(1 << 30) + 1, wst=(1 << 30) + 1) == UNS
    assert evict(c, out=cache(dtype=rkv.F16, K=2 * P, V=3 * P)) == INV
    assert evict(c, out=cache(dim_head=32, K=2 * P, V=3 * P)) == INV
    assert evict(c, out=cache(num_heads_kv=1, K=2 * P, V=3 * P)) == INV
    assert evict(c, out=cache(V=3 * P)) == INV                 # K in place, V elsewhere
    assert evict(c, out=cache(page_size=8)) == INV             # in place under another layout
    assert evict(c, batch=0) == OK


def test_decode_workspace_covers_every_window():
    """The workspace of max_len serves any sinks and window (a refusal would be
    RKV_ERR_WORKSPACE before anything is launched)."""
    b = ctypes.c_size_t(0)
    L = rkv.lib()
    assert L.rkv_paged_decode_workspace_size(4, 3, 64, 10, 1, 0, ctypes.byref(b)) == INV
    assert L.rkv_paged_decode_workspace_size(4, 2, 65, 10, 1, 0, ctypes.byref(b)) == UNS
    assert L.rkv_paged_decode_workspace_size(4, 2, 64, 10, 1, 0, None) == INV
    last = 0
    for n in list(range(0, 3000, 37)) + [12800, 12900, 131072]:
        assert L.rkv_paged_decode_workspace_size(24, 8, 128, n, 2, 0, ctypes.byref(b)) == OK
        assert b.value >= last, n
        last = b.value


def sink(Q=P, K=P, V=P, dt=rkv.BF16, lq=4, lk=8, batch=1, H=4, HK=2, D=64, qs=None, ks=None, sinks=0, window=0, O=P, os=None,
         ws=P, wb=256):
    r = lambda s: ctypes.byref(rkv._RowStrides(*s)) if s else None  # noqa: E731
    return rkv.lib().rkv_sink_attention(Q, K, V, dt, lq, lk, batch, H, HK, D, r(qs), r(ks), None, sinks, window, O, r(os), None,
                                        ws, wb, None)


def test_sink_attention_arguments():
    assert sink(dt=rkv.Q8_0) == INV and sink(dt=-1) == INV
    assert sink(lq=9) == INV and sink(lq=-1) == INV and sink(H=3) == INV and sink(HK=0) == INV and sink(batch=-1) == INV
    assert sink(sinks=-1) == INV and sink(window=-1) == INV
    assert sink(D=60) == UNS and sink(D=264) == UNS and sink(D=0) == INV
    for name in ("Q", "K", "V", "O"):
        assert sink(**{name: None}) == INV and sink(**{name: P + 8}) == INV
    assert sink(qs=(0, 512, 136)) == INV and sink(ks=(0, 8, 128)) == INV and sink(os=(0, 512, 64)) == INV
    assert sink(batch=2, qs=(64, 512, 128)) == INV
    assert sink(ws=None) == WS and sink(wb=8) == WS and sink(ws=P + 1) == WS
    assert sink(lq=0) == OK and sink(batch=0) == OK
    b = ctypes.c_size_t(0)
    size = rkv.lib().rkv_sink_attention_workspace_size
    assert size(rkv.BF16, 8, 8, 1, 4, 2, 64, None) == INV and size(rkv.BF16, 9, 8, 1, 4, 2, 64, ctypes.byref(b)) == INV
    assert size(rkv.BF16, 8, 8, 1, 4, 2, 60, ctypes.byref(b)) == UNS
    for dt, D in ((rkv.BF16, 64), (rkv.F16, 128), (rkv.F32, 128), (rkv.BF16, 256), (rkv.F32, 256)):
        assert size(dt, 4, 8, 1, 4, 2, D, ctypes.byref(b)) == OK and b.value >= 4
        # few queries over many keys: parts of the keys, whatever the window
        assert size(dt, 4, 100000, 1, 4, 2, D, ctypes.byref(b)) == OK and b.value > 4 * 4 * D * 4
        assert sink(dt=dt, D=D, lk=100000, window=0, wb=b.value - 1) == WS
        assert sink(dt=dt, D=D, lk=100000, window=99999, wb=256) == WS


def test_python_front_end_refuses_cpu_tensors():
    import torch
    K = torch.zeros((4, 2, 16, 64))
    with pytest.raises((TypeError, ValueError)):
        rkv.PagedCache(K, K, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        rkv.PagedCache(K, K[:, :1], torch.zeros((1, 2), dtype=torch.int32), None)


def test_evict_into_too_few_pages():
    """A destination without room for the rows that stay is refused: they would
    be lost while new_lens counts them."""
    c = cache()  # 32 tokens of a sequence, 16 stay
    assert evict(c, out=cache(K=2 * P, V=3 * P, table_stride=1, page_size=8, page_stride=2 * 8 * 128, head_stride=8 * 128)) == INV
    assert evict(c, budget=100, kst=100, max_len=100, wst=100, out=cache(K=2 * P, V=3 * P, table_stride=1)) == INV
