"""Calls of the paged-cache entry points that have nothing to do: host logic."""
import ctypes

import pytest

import rocketkv_b200 as rkv

P = 1 << 20  # stands for a device address: never followed


def _cache(**kw):
    f = dict(K=P, V=P, dtype=rkv.BF16, num_heads_kv=2, dim_head=64, page_size=16, num_pages=4, table_stride=2,
             page_stride=2 * 16 * 128, head_stride=16 * 128, token_stride=128, block_table=None, lens=None)
    f.update(kw)
    return ctypes.byref(rkv._PagedCache(**f))


def _calls(cache, batch):
    L = rkv.lib()
    return {
        "append": L.rkv_paged_append(cache, None, None, 1, batch, 256, 256, 128, None, None),
        "decode": L.rkv_paged_decode(None, 512, 4, cache, 32, batch, 0, 0, None, None, None, 0, None, 0, None),
        "evict": L.rkv_weight_evict(cache, None, 32, 32, batch, 16, 2, 2, None, None, None, 16, None, None),
        "evict to": L.rkv_weight_evict(cache, None, 32, 32, batch, 16, 2, 2, _cache(K=2 * P, V=3 * P), None, None, 16, None, None),
    }


def test_a_batch_without_a_sequence_needs_no_table_or_lengths():
    """An empty tensor has no address; the call has nothing to do."""
    assert set(_calls(_cache(), 0).values()) == {rkv.RKV_OK}
    assert set(_calls(_cache(), 1).values()) == {rkv.RKV_ERR_INVALID_ARG}
    assert set(_calls(_cache(block_table=P), 1).values()) == {rkv.RKV_ERR_INVALID_ARG}


@pytest.mark.parametrize("bad", [dict(dim_head=60), dict(K=P + 8), dict(dtype=9), dict(page_size=0)])
def test_what_else_is_wrong_is_still_refused(bad):
    assert rkv.RKV_OK not in _calls(_cache(**bad), 0).values()
