"""Plain 64-bit forms of the block-scaled 8-bit operators (numpy): what
aut_encode_scaled, aut_rms_norm_scaled and aut_gemm_scaled are tested against."""
import numpy as np

BLOCK = 128
E4M3, E5M2 = 0, 1
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
U = 2.0 ** -24  # half an ulp of FP32, relative


def code_values(code):
    """The value of each of the 256 codes: 4 exponent bits with bias 7 and 3
    fraction bits (one NaN magnitude, 0x7f), or 5 with bias 15 and 2 (exponent
    31: infinity for fraction 0, else NaN)."""
    bits, bias = (3, 7) if code == E4M3 else (2, 15)
    c = np.arange(256)
    exponent, fraction = (c & 0x7f) >> bits, c & ((1 << bits) - 1)
    v = np.where(exponent == 0, fraction * 2.0 ** (1 - bias - bits),
                 (1 + fraction / 2.0 ** bits) * 2.0 ** (exponent - bias))
    if code == E4M3:
        v[(c & 0x7f) == 0x7f] = np.nan
    else:
        v[(exponent == 31) & (fraction == 0)] = np.inf
        v[(exponent == 31) & (fraction != 0)] = np.nan
    return np.where(c >= 128, -v, v)


def round_to_code(q, code):
    """The value of the code nearest to q (ties to even, magnitudes above the
    largest value to it, what is not a number to NaN)."""
    q = np.asarray(q, np.float64)
    bits, low = (3, -6) if code == E4M3 else (2, -14)
    with np.errstate(invalid="ignore"):
        exponent = np.frexp(q)[1] - 1
        step = np.exp2(np.maximum(exponent, low).astype(np.float64) - bits)
        return np.clip(np.rint(q / step) * step, -LARGEST[code], LARGEST[code])


def _padded(x, block_rows):
    rows, columns = x.shape
    nr, nb = -(-rows // block_rows), -(-columns // BLOCK)
    full = np.zeros((nr * block_rows, nb * BLOCK), x.dtype)
    full[:rows, :columns] = x
    return full.reshape(nr, block_rows, nb, BLOCK)


def scales_of(x, code, block_rows):
    """scales[b, R] in the type of x (FP32 in: one rounded division)."""
    blocks = _padded(x, block_rows)
    largest = np.where(np.isfinite(blocks), np.abs(blocks), 0).max(axis=(1, 3))
    return np.maximum(largest / x.dtype.type(LARGEST[code]), x.dtype.type(2.0 ** -126)).T


def spread(scales, rows, columns, block_rows):
    """scales[b, R] as one scale per element."""
    return np.repeat(np.repeat(scales.T, block_rows, 0)[:rows], BLOCK, 1)[:, :columns]


def encode(x, code, block_rows):
    """(values of the codes, scales) of FP32 x, as the library defines them: the
    scale and the quotient each rounded once to FP32."""
    x = np.asarray(x, np.float32)
    scales = scales_of(x, code, block_rows)
    with np.errstate(invalid="ignore"):
        q = x / spread(scales, *x.shape, block_rows)
        q = np.where(np.isfinite(x), q, np.float32(np.nan))
    return round_to_code(q, code), scales


def rms_norm(x, residual, weight, eps):
    """(h, y) in 64 bits."""
    h = np.asarray(x, np.float64) + (0.0 if residual is None else np.asarray(residual, np.float64))
    with np.errstate(all="ignore"):
        y = h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + eps)
    return h, y * (1.0 if weight is None else np.asarray(weight, np.float64))


def norm_tolerance(columns):
    """Relative error bound of the kernels' y in FP32.  The sum of squares: at
    most columns / 32 terms in a thread's chain and 16 additions joining the
    threads, each within U (positive terms), so half of that in the root; the
    mean, eps and their rounding 3 U halved; the reciprocal root 4 U; h, its
    square (2 U halved), and two products 5 U."""
    return (0.5 * (columns / 32 + 16 + 3) + 4 + 5) * U


def check_codes(values, scales, y, code, block_rows, tolerance):
    """Values and scales of codes against y in 64 bits, y within `tolerance`
    (relative): the scale within it plus its own rounding, each code one that a
    y within it rounds to."""
    want = scales_of(y, code, block_rows)
    np.testing.assert_allclose(scales, want, rtol=tolerance + 2 * U, atol=0)
    s = spread(scales.astype(np.float64), *y.shape, block_rows)
    fine = np.isfinite(y)
    assert np.array_equal(np.isnan(values), ~fine)
    q = np.where(fine, y, 0) / s
    width = tolerance + 4 * U
    a, b = round_to_code(q * (1 - width), code), round_to_code(q * (1 + width), code)
    v = np.where(fine, values, 0)
    assert np.all((np.minimum(a, b) <= v) & (v <= np.maximum(a, b)))


def gemm(a, a_scales, b, b_scales):
    """(product, sum of magnitudes) in 64 bits of code values and scales."""
    with np.errstate(all="ignore"):
        a = a * spread(a_scales.astype(np.float64), *a.shape, 1)
        b = b * spread(b_scales.astype(np.float64), *b.shape, BLOCK)
        return a @ b.T, np.abs(a) @ np.abs(b).T


def gemm_tolerance(k):
    """Error bound over the sum of magnitudes: within a block of 128 each of the
    instruction's additions is within 2 U (whether it rounds or truncates), each
    block's product with the two scales and its addition within 4 U of it, the
    additions over the blocks within U each, the joins of partial sums 16 U."""
    return (2 * BLOCK + 4 + -(-k // BLOCK) + 16) * U

