"""Rotary positions: the frequencies' fixed point and what the entry points
refuse; host logic only, nothing is launched."""
import ctypes
import math
from fractions import Fraction

import pytest

import rocketkv_b200 as rkv

INV, UNS, OK = rkv.RKV_ERR_INVALID_ARG, rkv.RKV_ERR_UNSUPPORTED, rkv.RKV_OK
P = 1 << 20  # stands for a device address: never followed


def _freqs(values):
    n = len(values)
    out = (ctypes.c_uint64 * max(1, n))()
    st = rkv.lib().rkv_rotary_frequencies((ctypes.c_double * max(1, n))(*values), n, out)
    return st, list(out)[:n]


# 2 pi to 40 digits
TWO_PI = Fraction("6.283185307179586476925286766559005768394")


def test_frequencies_are_turns_in_64_bits():
    """f / 2 pi modulo a turn.  The quotient is formed with 64 significant bits
    or more (2^-63 of it, from the rounded 2 pi and the rounded quotient), then
    rounded to a step."""
    values = [1.0, 0.5, 500000.0 ** -0.9, 1e-9, 6.0, 7.0, 0.0, -0.25, 1234.5]
    st, got = _freqs(values)
    assert st == OK
    for f, g in zip(values, got):
        want = Fraction(f) / TWO_PI * 2 ** 64
        off = (Fraction(g) - want) % 2 ** 64
        off = min(off, 2 ** 64 - off)
        assert off <= Fraction(1, 2) + abs(want) / 2 ** 62, f
    assert got[6] == 0
    # the angle of a far position: exact modulo a turn
    p = 2 ** 31 - 1
    want = (Fraction(1.0) / TWO_PI * p) % 1
    off = (Fraction(got[0] * p % 2 ** 64, 2 ** 64) - want) % 1
    assert min(off, 1 - off) < Fraction(1, 2 ** 31)


def test_frequencies_refused():
    L = rkv.lib()
    one = (ctypes.c_double * 1)(1.0)
    out = (ctypes.c_uint64 * 1)()
    assert L.rkv_rotary_frequencies(None, 1, out) == INV and L.rkv_rotary_frequencies(one, 1, None) == INV
    assert L.rkv_rotary_frequencies(one, -1, out) == INV
    for bad in (math.nan, math.inf, -math.inf):
        assert _freqs([1.0, bad])[0] == INV
    assert _freqs([])[0] == OK


def _rotary(**kw):
    f = dict(freqs=P, axes=None, pairs=32, num_axes=1, interleaved=0)
    f.update(kw)
    return rkv._Rotary(**f)


def _strides(s):
    return None if s is None else ctypes.byref(rkv._RowStrides(*s))


def rotate(r, pos=P, q=P, qo=P, H=4, k=P, ko=P, HK=2, dt=rkv.BF16, D=64, n=8, B=1, qs=None, qos=None, ks=None, kos=None):
    return rkv.lib().rkv_rotate(ctypes.byref(r) if r else None, pos, q, qo, H, k, ko, HK, dt, D, n, B, _strides(qs), _strides(qos),
                                _strides(ks), _strides(kos), None)


def _cache(**kw):
    f = dict(K=P, V=P, dtype=rkv.BF16, num_heads_kv=2, dim_head=64, page_size=16, num_pages=4, table_stride=2,
             page_stride=2 * 16 * 128, head_stride=16 * 128, token_stride=128, block_table=P, lens=P)
    f.update(kw)
    return rkv._PagedCache(**f)


def append(c, r, pos=None, k=P, v=P, ks=None, n=1, B=1, n_new=None, q=P, qs=None, qo=P, qos=None, H=4):
    return rkv.lib().rkv_paged_append_rotated(ctypes.byref(c) if c else None, ctypes.byref(r) if r else None, pos, k, v, _strides(ks), n,
                                              B, n_new, q, _strides(qs), qo, _strides(qos), H, None)


@pytest.mark.parametrize("kw", [dict(pairs=0), dict(pairs=33), dict(pairs=-1), dict(num_axes=0), dict(freqs=None), dict(freqs=P + 4)])
def test_bad_rotaries(kw):
    assert rotate(_rotary(**kw)) == INV and append(_cache(), _rotary(**kw)) == INV


def test_rotate_arguments():
    r = _rotary()
    assert rotate(None) == INV and rotate(_rotary(num_axes=257)) == UNS
    assert rotate(r, dt=rkv.Q8_0) == INV and rotate(r, dt=9) == INV
    assert rotate(r, D=60) == INV and rotate(r, D=68) == UNS and rotate(r, D=264) == UNS
    assert rotate(r, H=-1) == INV and rotate(r, HK=-1) == INV and rotate(r, n=-1) == INV and rotate(r, B=-1) == INV
    for name in ("pos", "q", "qo", "k", "ko"):
        assert rotate(r, **{name: None}) == INV
    for name in ("q", "qo", "k", "ko"):
        assert rotate(r, **{name: P + 1}) == INV
    assert rotate(r, dt=rkv.F32, q=P + 2) == INV
    assert rotate(r, qs=(0, -128, 128)) == INV and rotate(r, qs=(0, 1024, 129)) == INV
    assert rotate(r, qos=(0, 1024, 64)) == INV and rotate(r, qos=(0, 0, 128)) == INV  # rows that are written would meet
    assert rotate(r, B=2, kos=(64, 1024, 128)) == INV
    assert rotate(r, B=70000) == UNS
    assert rotate(r, n=0) == OK and rotate(r, B=0) == OK
    assert rotate(r, H=0, HK=0, q=None, qo=None, k=None, ko=None) == OK


def test_append_arguments():
    r, c = _rotary(), _cache()
    assert append(None, r) == INV and append(c, None) == INV
    assert append(_cache(dim_head=60), r) == UNS and append(_cache(lens=None), r) == INV and append(_cache(dtype=rkv.Q8_0), r) == INV
    assert append(c, r, n=-1) == INV and append(c, r, B=-1) == INV and append(c, r, H=-1) == INV
    assert append(c, r, k=None) == INV and append(c, r, v=None) == INV and append(c, r, q=None) == INV and append(c, r, qo=None) == INV
    assert append(c, r, k=P + 1) == INV and append(c, r, qo=P + 1) == INV
    assert append(c, r, n=2, ks=(0, 128, 129)) == INV and append(c, r, ks=(0, -128, 128)) == INV
    assert append(c, r, n=2, qos=(0, 128, 128 - 16)) == INV
    assert append(c, r, B=70000) == UNS
    assert append(c, r, n=0) == OK and append(c, r, B=0) == OK


def test_python_front_end():
    import torch
    f = torch.ones(8, dtype=torch.float64)
    for bad in (dict(inv_freq=f, dim_head=8), dict(inv_freq=f[:0], dim_head=64), dict(inv_freq=f[None], dim_head=64),
                dict(inv_freq=f, dim_head=64, axes=[0] * 7), dict(inv_freq=f, dim_head=64, axes=[-1] * 8),
                dict(inv_freq=f, dim_head=64, axes=[2] * 8, num_axes=2), dict(inv_freq=f, dim_head=64, axes=[256] * 8)):
        with pytest.raises(ValueError):
            rkv.Rotary(device="cpu", **bad)
    with pytest.raises(rkv.RkvError):
        rkv.Rotary(f * math.inf, 64, device="cpu")
    with pytest.raises(ValueError):
        rkv.rotate(None, None, None, None)
