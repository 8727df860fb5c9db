"""The block-scaled operators at the limits of their definition."""
import numpy as np
import pytest

import scaled_ref as ref
from test_gpu_scaled import FP32, check_gemm, check_norm, operand, run_gemm, run_norm, values

pytestmark = pytest.mark.gpu

INFINITY = 0x7C  # E5M2


# one token, few rows, tiles whose k is cut into 2 or 4 parts on 32 and 64 columns,
# uncut tiles of 32, 64, 128 and 256 columns, rows on any boundary (stride 1)
INFINITE = [(1, 300, 5120, 0), (12, 300, 5120, 0), (64, 1024, 5120, 0), (32, 1024, 5120, 0),
            (87, 256, 2333, 0), (100, 1000, 3000, 0), (150, 300, 2304, 0), (33, 520, 640, 0),
            (300, 10300, 2000, 0), (300, 6500, 1999, 0), (20, 300, 2000, 1), (70, 300, 2000, 1)]


@pytest.mark.parametrize("size", INFINITE)
@pytest.mark.parametrize("side", ["a", "b"])
def test_an_infinite_code_gives_an_infinite_result(ws, size, side):
    """One infinity in each block of k, each in a row of its own, against codes
    that are not zero: its row (or column) is infinite with the sign of the
    product, all others are as without it."""
    m, n, k, off = size
    blocks = -(-k // 128)
    a, sa = operand(m, k, ref.E5M2, 1, 5)
    b, sb = operand(n, k, ref.E5M2, 128, 6)
    a[a & 0x7F == 0] = 0x3C
    b[b & 0x7F == 0] = 0x3C
    layout = dict(a_stride=k + off + k % 2, b_stride=k + off + k % 2) if off else {}
    codes = (ref.E5M2, ref.E5M2)
    clean = run_gemm(ws, a, sa, b, sb, *codes, FP32, **layout)
    check_gemm(clean, a, sa, b, sb, *codes, FP32)
    own, other = (a, b) if side == "a" else (b, a)
    for first in range(0, blocks, own.shape[0]):
        marked = own.copy()
        want = clean.copy() if side == "a" else clean.T.copy()
        for row, block in enumerate(range(first, min(blocks, first + own.shape[0]))):
            at = min(128 * block + 17 * block % 128, k - 1)
            marked[row, at] = INFINITY | 0x80 * (block % 2)
            sign = np.where((other[:, at] ^ marked[row, at]) & 0x80, -1.0, 1.0)
            want[row] = sign * np.inf
        pair = (marked, sa, b, sb) if side == "a" else (a, sa, marked, sb)
        got = run_gemm(ws, *pair, *codes, FP32, **layout)
        np.testing.assert_array_equal(got, want if side == "a" else want.T)


# of each of the product's kernels: one token, few rows, a long k shared by a
# cluster, tiles of 32 (cut and uncut), 64, 128 and 256 columns, any boundary
RANGES = [(1, 300, 700, 0), (8, 40, 9000, 0), (12, 300, 700, 0), (64, 1024, 5120, 0),
          (33, 520, 640, 0), (129, 700, 3000, 0), (150, 3000, 700, 0), (300, 10300, 700, 0),
          (300, 6500, 700, 0), (9, 300, 700, 1), (70, 300, 700, 1)]


def large_codes(rows, columns, seed):
    """E5M2 codes of magnitudes 2^12 to 57344."""
    rng = np.random.default_rng(seed)
    return (rng.integers(0x6C, 0x7C, (rows, columns)) | 0x80 * rng.integers(0, 2, (rows, columns))
            ).astype(np.uint8)


def small_codes(rows, columns, seed):
    """E4M3 codes of magnitudes 0 to 3 * 2^-9."""
    rng = np.random.default_rng(seed)
    return (rng.integers(0, 4, (rows, columns)) | 0x80 * rng.integers(0, 2, (rows, columns))
            ).astype(np.uint8)


def scales_near(shape, exponents, seed):
    rng = np.random.default_rng(seed)
    e = rng.choice(exponents, size=shape) if np.ndim(exponents) else exponents
    return ((1 + rng.random(shape)) * 2.0 ** e).astype(np.float32)


def layout_of(k, off):
    return dict(a_stride=k + off + k % 2, b_stride=k + off + k % 2) if off else {}


def check_products_first(got, a, sa, b, sb, a_code, b_code):
    """The result where the two scales are multiplied first, in FP32: within
    gemm_tolerance of the sum in 64 bits and, for terms below the normal range,
    half of the smallest number for each block of k."""
    av, bv = ref.code_values(a_code)[a], ref.code_values(b_code)[b]
    k = a.shape[1]
    want, size = np.zeros(got.shape), np.zeros(got.shape)
    for block in range(-(-k // 128)):
        c = slice(128 * block, 128 * (block + 1))
        s = np.outer(sa[block], np.repeat(sb[block], 128)[:b.shape[0]]).astype(np.float32)
        want += (av[:, c] @ bv[:, c].T) * s
        size += (np.abs(av[:, c]) @ np.abs(bv[:, c]).T) * np.abs(s)
    bound = ref.gemm_tolerance(k) * size + -(-k // 128) * 2.0 ** -150
    low, high = (want - bound).astype(np.float32), (want + bound).astype(np.float32)
    assert np.all((low <= got) & (got <= high)), np.max(np.abs(got - want) / (bound + 1e-300))


@pytest.mark.parametrize("size", RANGES)
@pytest.mark.parametrize("exponents", [(-75, -75), (-70, -70), (-126, -10), (-126, -26),
                                       ((-90, -60, -20), (-60, -70))])
def test_products_of_scales_below_the_normal_range(ws, size, exponents):
    """The scales are multiplied first, whatever the kernel; zeros stay zeros."""
    m, n, k, off = size
    a, b = large_codes(m, k, 1), large_codes(n, k, 2)
    sa = scales_near((-(-k // 128), m), exponents[0], 3)
    sb = scales_near((-(-k // 128), -(-n // 128)), exponents[1], 4)
    b[5] = 0
    got = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E5M2, FP32, **layout_of(k, off))
    check_products_first(got, a, sa, b, sb, ref.E5M2, ref.E5M2)
    assert (got[:, 5] == 0).all()


@pytest.mark.parametrize("size", RANGES)
def test_products_of_scales_above_the_largest_value(ws, size):
    """Infinite: so is the result with the sign of the sums, and NaN where a sum is 0."""
    m, n, k, off = size
    a, b = np.full((m, k), 0x38, np.uint8), np.full((n, k), 0x38, np.uint8)
    sa = np.ones((-(-k // 128), m), np.float32)
    sb = np.full((-(-k // 128), -(-n // 128)), 2.0 ** 40, np.float32)
    sa[0] = 2.0 ** 100
    b[1], b[5] = 0xB8, 0
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32, **layout_of(k, off))
    columns = np.arange(n)
    assert (got[:, 1] == -np.inf).all() and np.isnan(got[:, 5]).all()
    assert (got[:, (columns != 1) & (columns != 5)] == np.inf).all()


@pytest.mark.parametrize("size", RANGES)
def test_rows_of_zeros_with_the_smallest_scale(ws, size):
    m, n, k, off = size
    a, sa = operand(m, k, ref.E4M3, 1, 5)
    b, sb = operand(n, k, ref.E4M3, 128, 6)
    sa[:, ::2], a[::2] = 2.0 ** -126, 0
    sb[0] = 2.0 ** -120
    sb[-1] = 2.0 ** 127
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32, **layout_of(k, off))
    assert (got[::2] == 0).all()


@pytest.mark.parametrize("size", RANGES)
def test_scales_that_are_zero_or_not_finite(ws, size):
    """A scale counts in its own row (or 128 columns) alone."""
    m, n, k, off = size
    a, sa = operand(m, k, ref.E4M3, 1, 5)
    b, sb = operand(n, k, ref.E4M3, 128, 6)
    a[a & 0x7F == 0] = 0x38
    b[b & 0x7F == 0] = 0x38
    sa[:, 0] = 0
    if m > 5:
        sa[1, 1], sa[2, 2], sa[3, 3] = np.nan, np.inf, -sa[3, 3]
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32, **layout_of(k, off))
    assert (got[0] == 0).all()
    if m > 5:
        assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any()
        rest = [i for i in range(m) if i not in (1, 2)]
        check_gemm(got[rest], a[rest], sa[:, rest], b, sb, ref.E4M3, ref.E4M3, FP32)
    if sb.shape[1] > 1:
        sa[:] = 1
        sb[1, 1] = np.nan
        got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32, **layout_of(k, off))
        inside = np.arange(n) // 128 == 1
        assert np.isnan(got[:, inside]).all() and np.isfinite(got[:, ~inside]).all()


@pytest.mark.parametrize("columns", [200, 512, 5001, 16392])
def test_norm_of_rows_beyond_the_range_of_their_squares(ws, columns):
    """Zeros where the sum of squares overflows; just below, values as any other."""
    x = values(4, columns, 3, spread=0.1)
    x[1] *= 2.0 ** 70
    x[2] = 2.0 ** 54
    got, after = run_norm(ws, x, None, None, 1e-5, FP32, ref.E4M3, into="new")
    assert (got[0][1] == 0).all() and (got[1][:, 1] == np.float32(2.0 ** -126)).all()
    np.testing.assert_array_equal(after, x.astype(np.float32))
    rest = [0, 2, 3]
    check_norm((got[0][rest], got[1][:, rest]), after[rest], x[rest], None, None, 1e-5, FP32,
               ref.E4M3)
