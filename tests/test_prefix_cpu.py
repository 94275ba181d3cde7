"""What the shared-prefix decode refuses, and its size query: host logic only,
nothing is launched."""
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


def decode(c, Q=P, qs=4 * 128, H=4, max_len=32, batch=1, starts=P, tokens=P, groups=1, O=P, lse=None, ws=P, wb=1 << 40):
    return rkv.lib().rkv_prefix_decode(Q, qs, H, ctypes.byref(c) if c else None, max_len, batch, starts, tokens, groups, O, lse, ws, wb, None)


def size(dt=rkv.BF16, H=24, HK=8, D=128, max_len=4096, batch=8, groups=1):
    b = ctypes.c_size_t(0)
    return rkv.lib().rkv_prefix_decode_workspace_size(dt, H, HK, D, max_len, batch, groups, ctypes.byref(b)), b.value


@pytest.mark.parametrize("kw,want", [
    (dict(dtype=rkv.Q8_0), INV), (dict(num_heads_kv=0), INV), (dict(page_size=0), INV), (dict(dim_head=60), UNS), (dict(dim_head=264), UNS),
    (dict(K=P + 8), INV), (dict(token_stride=136), INV), (dict(head_stride=64), INV), (dict(V=None), INV), (dict(block_table=None), INV),
    (dict(lens=None), INV)])
def test_bad_caches(kw, want):
    assert decode(cache(**kw)) == want


def test_arguments():
    c = cache()
    assert decode(None) == INV
    assert decode(c, H=3) == INV and decode(c, H=0) == INV and decode(c, max_len=-1) == INV and decode(c, batch=-1) == INV
    assert decode(c, groups=-1) == INV and decode(c, max_len=(1 << 30) + 1) == UNS and decode(c, H=2 * 1025) == UNS
    assert decode(c, groups=(1 << 24) + 1) == UNS and decode(c, batch=1 << 29) == UNS
    assert decode(c, Q=None) == INV and decode(c, Q=P + 8) == INV and decode(c, O=None) == INV and decode(c, O=P + 8) == INV
    assert decode(c, batch=2, qs=8) == INV and decode(c, batch=2, qs=4 * 128 + 8) == INV
    assert decode(c, starts=None) == INV and decode(c, tokens=None) == INV
    assert decode(c, ws=None) == WS and decode(c, ws=P + 4) == WS and decode(c, wb=8) == WS
    assert decode(c, groups=0, starts=None, tokens=None, wb=8) == WS  # no groups need no arrays
    assert decode(c, batch=0, Q=None, O=None, starts=None, tokens=None, ws=None) == OK


def test_sizes():
    assert size(dt=rkv.Q8_0)[0] == INV and size(HK=5)[0] == INV and size(D=0)[0] == INV and size(D=60)[0] == UNS
    assert size(batch=-1)[0] == INV and size(groups=-1)[0] == INV and size(max_len=(1 << 30) + 1)[0] == UNS
    assert rkv.lib().rkv_prefix_decode_workspace_size(rkv.BF16, 24, 8, 128, 4096, 8, 1, None) == INV
    for dt in (rkv.BF16, rkv.F16, rkv.F32):
        for D in (8, 64, 128, 136, 256):
            for batch in (0, 1, 64, 300):
                for groups in (0, 1, 7):
                    for n in (0, 1, 1000, 131072, 1 << 30):
                        st, b = size(dt=dt, D=D, batch=batch, groups=groups, max_len=n)
                        assert st == OK and b >= 256
                        # at least one part of every row, (m, l) and fp32 output
                        assert b >= batch * 24 * (8 + 4 * D)
                        # and no more than a few parts where the batch is large
                        assert b <= 256 * 1024 + batch * 24 * (8 + 4 * D) * 200 + 148 * 256 * (8 + 4 * D)


def test_python_front_end_needs_the_type():
    import torch
    with pytest.raises((TypeError, rkv.RkvError)):
        rkv.PrefixDecoder(24, 8, 128, 100, 2, torch.int8, "cpu")
    with pytest.raises(rkv.RkvError):
        rkv.PrefixDecoder(24, 7, 128, 100, 2, torch.bfloat16, "cpu")
