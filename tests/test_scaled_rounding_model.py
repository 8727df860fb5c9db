"""The arithmetic by which the kernels divide by a scale (scaled_device.cuh), in
exact integers: the reciprocal over every fraction that a scale can have, and the
quotients beside the midpoints that decide a code."""
from fractions import Fraction
import math

import numpy as np
import pytest

import scaled_ref as ref
from test_gpu_scaled_rounding import quotients_beside_a_midpoint

NEXT = (-1, 0, 1)  # ulp that the hardware's approximation may lie beside the nearest value


def up32(x):
    """FP32 values of extended-precision x, rounded up."""
    f = x.astype(np.float32)
    return np.where(f.astype(np.longdouble) < x, np.nextafter(f, np.float32(9)), f)


@pytest.mark.parametrize("step", NEXT)
def test_the_reciprocal_is_rounded_down(step):
    s = np.arange(1 << 23, 1 << 24, dtype=np.int64)  # scale s 2^-23
    down, rest = np.divmod(np.int64(1 << 47), s)  # 1 / scale in units of 2^-24
    r = down + (2 * rest > s) + step
    e = (((1 << 47) - s * r).astype(np.float64) * 2.0 ** -47).astype(np.float32)  # one FMA
    e = e.astype(np.longdouble)
    fraction, exponent = np.frexp(up32(e + e * e))
    t = (fraction.astype(np.float64) * 2.0 ** 24).astype(np.int64)  # t 2^(exponent - 24)
    inverse = r + ((r * t) >> np.minimum(24 - exponent.astype(np.int64), 62))
    np.testing.assert_array_equal(inverse, down)


def rounded(x, up=False, to_zero=False):
    """A fraction that is not negative as FP32 (normal range), to nearest even."""
    if x == 0:
        return Fraction(0)
    e = math.floor(math.log2(x.numerator) - math.log2(x.denominator))
    e += (Fraction(2) ** (e + 1) <= x) - (Fraction(2) ** e > x)
    unit = Fraction(2) ** (e - 23)
    n, left = divmod(x, unit)
    if not to_zero:
        half = unit / 2
        n += left > 0 if up else left > half or (left == half and n % 2)
    return n * unit


@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
def test_quotients_beside_a_midpoint_are_rounded_once(code):
    count = 0
    for s, quotients in quotients_beside_a_midpoint(code, furthest=32):
        s = Fraction(s)
        inverse = rounded(1 / s, to_zero=True)
        e = 1 - s * inverse
        assert e >= 0 and rounded(e) == e
        rest = rounded(inverse * rounded(e + e * e, up=True), to_zero=True)
        for x in map(Fraction, quotients):
            assert rounded(x * inverse + rounded(x * rest)) == rounded(x / s)
            count += 1
    assert count > 1000
