"""The block-scaled operators at the limits of their definition."""
import numpy as np
import pytest

import scaled_ref as ref
from test_gpu_scaled import FP32, check_gemm, operand, run_gemm

pytestmark = pytest.mark.gpu

INFINITY = 0x7C  # E5M2


# one token, few rows, tiles whose k is cut into 2 or 4 parts on 32 and 64 columns,
# uncut tiles of 32, 64, 128 and 256 columns, rows on any boundary (stride 1)
INFINITE = [(1, 300, 5120, 0), (12, 300, 5120, 0), (64, 1024, 5120, 0), (32, 1024, 5120, 0),
            (87, 256, 2333, 0), (100, 1000, 3000, 0), (150, 300, 2304, 0), (33, 520, 640, 0),
            (300, 10300, 2000, 0), (129, 9000, 1500, 0), (20, 300, 2000, 1), (70, 300, 2000, 1)]


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
