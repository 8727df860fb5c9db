"""Codes are those of the quotient x / scale rounded once to FP32 and once to the
code, at the quotients where an error of one part in 2^46 shows, and with the sign
of a zero."""
from fractions import Fraction

import numpy as np
import pytest

import scaled_ref as ref
from test_gpu_scaled import BF16, FP16, FP32, rounded, run_encode, values

pytestmark = pytest.mark.gpu


def quotients_beside_a_midpoint(code, furthest=8):
    """(s, [x, ...]): s in [1, 2), each x / s within `furthest` parts in 2^48 of the
    midpoint between a tie of two codes and a neighbour of it in FP32.  On one side
    of that midpoint FP32 rounds to the tie, which goes to the even code, on the
    other to the neighbour, which does not.

    With the midpoint M 2^e, M odd of 25 bits, and s = S 2^-23, x = X 2^j:
    X 2^q = M S + d for a small d, so S = -d / M modulo 2^q."""
    v = ref.code_values(code)
    v = np.unique(np.abs(v[np.isfinite(v)]))
    found = {}
    for t in ((v[1:] + v[:-1]) / 2).astype(np.float32):
        for beside in (np.nextafter(t, np.float32(0)), np.nextafter(t, np.float32(1e9))):
            middle = (Fraction(float(t)) + Fraction(float(beside))) / 2
            m, e = middle.numerator, -(middle.denominator.bit_length() - 1)
            while m % 2 == 0:
                m, e = m // 2, e + 1
            assert m.bit_length() == 25
            for q in (24, 25):
                inverse = pow(m, -1, 1 << q)
                for d in range(-furthest, furthest + 1):
                    s = -d * inverse % (1 << q)
                    if d == 0 or not 1 << 23 <= s < 1 << 24:
                        continue
                    x = (m * s + d) >> q
                    if 1 << 23 <= x < 1 << 24:
                        found.setdefault(s, set()).add(float(Fraction(x << q) * Fraction(2) ** (e - 23)))
    return [(s * 2.0 ** -23, sorted(x)) for s, x in sorted(found.items())]


def blocks_of(code, exponent):
    """One block of 128 to each scale s 2^exponent: the value that makes it the
    scale, then quotients of both signs beside midpoints; those that FP32 cannot
    hold are left out."""
    rows = []
    for s, quotients in quotients_beside_a_midpoint(code):
        scale = np.float32(s * 2.0 ** exponent)
        largest = np.float32(float(scale) * ref.LARGEST[code])
        if np.float32(largest / np.float32(ref.LARGEST[code])) != scale:
            continue
        x = np.array(quotients) * 2.0 ** exponent
        x = x[(x.astype(np.float32) == x) & (x <= largest)]
        row = np.resize(np.concatenate([x, -x]) if x.size else np.zeros(1), 128)
        row[0] = largest
        rows.append(row)
    return np.array(rows)


def check_bits(got, x, code, block_rows):
    """Equal to the definition, signs of zeros among them."""
    want, scales = ref.encode(x, code, block_rows)
    np.testing.assert_array_equal(got[1], scales)
    np.testing.assert_array_equal(got[0], want)
    number = ~np.isnan(want)
    np.testing.assert_array_equal(np.signbit(got[0])[number], np.signbit(want)[number])


@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
@pytest.mark.parametrize("exponent", [-126, -110, -60, 0, 60, 90, 99, 100, 101, 105, 110])
def test_quotients_beside_a_tie(ws, code, exponent):
    x = blocks_of(code, exponent)
    assert x.shape[0] > 20
    check_bits(run_encode(ws, x, FP32, code, 1), x.astype(np.float32), code, 1)
    # the same by tiles: a block of 128 rows to each scale
    x = np.repeat(x[:40], 128, 0)
    check_bits(run_encode(ws, x, FP32, code, 128), x.astype(np.float32), code, 128)
    # and off 16-byte boundaries
    x = np.concatenate([x[::128], x[::128]], 1)
    check_bits(run_encode(ws, x, FP32, code, 1, x_stride=257, stride=259, offset=1),
               x.astype(np.float32), code, 1)


@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
@pytest.mark.parametrize("type", [FP32, BF16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_large_scales(ws, code, type, block_rows):
    """Blocks of values up to 2^128 beside blocks of small ones, and both in one."""
    x = values(384, 700, 3)
    x[:, 128:256] *= 2.0 ** 120
    x[130:, 300:500] *= 2.0 ** 104
    x[:, 600:] *= np.exp2(np.random.default_rng(4).integers(-120, 110, (384, 100)))
    x[3, 140], x[200, 140] = np.inf, -np.inf
    x = rounded(np.clip(x, -3e38, 3e38, where=np.isfinite(x), out=x), type)
    check_bits(run_encode(ws, x, type, code, block_rows), x, code, block_rows)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("columns", [512, 509])
def test_the_sign_of_a_zero(ws, type, code, block_rows, columns):
    """Zeros of both signs, and values that round to zero, beside ordinary values
    over many scales."""
    x = values(300, columns, 7) * np.exp2(np.arange(300) % 9)[:, None]
    rng = np.random.default_rng(8)
    x[rng.random(x.shape) < 0.2] = 0.0
    x[rng.random(x.shape) < 0.2] = -0.0
    x[:, 5] = -6e-8
    x = rounded(x, type)
    check_bits(run_encode(ws, x, type, code, block_rows), x, code, block_rows)
