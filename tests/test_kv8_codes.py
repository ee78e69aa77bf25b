"""The rounding of bf16 rows to the 8-bit cache's codes, every pair of mantissas: the
kernel's fp32 steps, restated in numpy, against exact arithmetic in integers.

A code is RNE(127 x / a).  The kernel takes x (127 / a) in fp32, rounds its bits to twenty
(add 8, clear the last four) and adds 2^23 + 2^22 + 128, whose sum's low byte is the code + 128.  Rows
whose largest magnitude is below 2^-100 are multiplied by 2^64 first."""
import numpy as np
import pytest


def kernel_codes(x, a):
    """x, a: float32 values of bf16 (0 < x <= a)."""
    f = np.float32
    k = np.where(a < f(2.0 ** -100), f(2.0 ** 64), f(1.0)).astype(f)
    x, a = (x * k).astype(f), (a * k).astype(f)
    inv = (f(127.0) / a).astype(f)
    t = (x * inv).astype(f).view(np.uint32)
    t = ((t + np.uint32(8)) & np.uint32(0xfffffff0)).view(f)
    return ((t + f(12582912.0 + 128.0)).astype(f).view(np.uint32) & 255).astype(np.int64) - 128


def exact_codes(mx, ma, gap):
    """RNE(127 mx / (ma 2^gap)) of whole numbers."""
    num, den = 127 * mx, ma << gap
    code, rest = num // den, 2 * (num % den)
    return code + ((rest > den) | ((rest == den) & (code % 2 == 1)))


@pytest.mark.parametrize("exponent", [-133, -126, -101, -100, -60, 0, 60, 119])
def test_every_pair_of_mantissas(exponent):
    """a = ma 2^exponent, x = mx 2^(exponent - gap), mantissas of eight bits; from
    a gap of 9 on a code is 0.  Subnormal rows (exponents below -126 here) have
    fewer bits: mantissas from 1, no gap."""
    subnormal = exponent < -126
    ma, mx = np.meshgrid(np.arange(1 if subnormal else 128, 256), np.arange(1 if subnormal else 128, 256), indexing="ij")
    for gap in range(1 if subnormal else 11):
        keep = mx <= (ma << gap)
        a = np.ldexp(ma[keep].astype(np.float64), exponent).astype(np.float32)
        x = np.ldexp(mx[keep].astype(np.float64), exponent - gap)
        if not subnormal and exponent - gap < -133:
            continue                                    # not a bf16 value
        x = x.astype(np.float32)
        assert (x.view(np.uint32) & 0xffff == 0).all() and (a.view(np.uint32) & 0xffff == 0).all()
        want = exact_codes(mx[keep].astype(np.int64), ma[keep].astype(np.int64), gap)
        assert np.array_equal(kernel_codes(x, a), want)
        assert np.array_equal(kernel_codes(-x, a), -want)
        assert gap < 9 or not want.any()
