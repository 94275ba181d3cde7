"""Frequencies of a rotation as fractions of a turn: the nearest step of 2^-64
turns whatever the radians, or a refusal.  Host logic only."""
import ctypes
import math
from fractions import Fraction

import pytest

import rocketkv_b200 as rkv


def _pi(bits):
    """floor(pi 2^bits), by Machin's formula: 16 atan(1/5) - 4 atan(1/239)."""
    one = 1 << (bits + 32)

    def atan(n):
        total, x, k = 0, one // n, 1
        while x:
            total += x // k if k % 4 == 1 else -(x // k)
            x //= n * n
            k += 2
        return total

    return (16 * atan(5) - 4 * atan(239)) >> 32


TWO_PI = Fraction(2 * _pi(600), 1 << 600)


def _freqs(values):
    n = len(values)
    out = (ctypes.c_uint64 * n)()
    return rkv.lib().rkv_rotary_frequencies((ctypes.c_double * n)(*values), n, out), list(out)


VALUES = [1.0, 0.1, 3.0, math.pi, 2 * math.pi, 7.0, 100.0, 1234.5, 1e6 + 0.1, 123456789.125, 1e9, 2.0 ** 32 + 1, 1e12 + 0.25, 1e15, 2.0 ** 53 + 2,
          1e18, 2.0 ** 63, math.nextafter(2.0 ** 64, 0.0), 6381956970095103.0 * 2.0 ** 9, 1e-3, 1e-19, 2.0 ** -62, 2.0 ** -64, 1e-25, 1e-300, 5e-324, 0.0]


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_nearest_step(sign):
    """Off by half a step of 2^-64 turns: a far position's angle, 2^31 of them,
    by 2^-34 turns."""
    values = [sign * v for v in VALUES]
    st, got = _freqs(values)
    assert st == rkv.RKV_OK
    for f, g in zip(values, got):
        want = Fraction(f) / TWO_PI * 2 ** 64
        off = (Fraction(g) - want) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 2 ** 40), f


def test_pi_is_pi():
    assert abs(TWO_PI / 2 - Fraction("3.14159265358979323846264338327950288419716939937510582097494459")) < Fraction(1, 10 ** 61)


def test_radians_that_are_no_angle_are_refused():
    for bad in (2.0 ** 64, -(2.0 ** 64), 1e20, 1e300, -1e308, math.inf, -math.inf, math.nan):
        assert _freqs([1.0, bad])[0] == rkv.RKV_ERR_INVALID_ARG, bad
    import torch
    with pytest.raises(rkv.RkvError):
        rkv.Rotary(torch.tensor([1e30], dtype=torch.float64), 64, device="cpu")
