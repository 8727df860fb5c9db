"""The block-scaled 8-bit operators (aut_encode_scaled, aut_rms_norm_scaled,
aut_gemm_scaled) against their plain 64-bit forms, and their refusals."""
import numpy as np
import pytest
import torch

import scaled_ref as ref
from accessor_universal_test_b200 import _lib

pytestmark = pytest.mark.gpu

FP32, BF16, FP16 = 0, 1, 2
TORCH = {FP32: torch.float32, BF16: torch.bfloat16, FP16: torch.float16}
GUARD = 0x5A  # what stands around the outputs


def rounded(x, type):
    """x rounded to `type`, as float32 numpy."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(TORCH[type]).float().numpy()


def device_matrix(x, type, stride, offset=0):
    """x on the device with a row stride and `offset` elements before it; the
    elements between rows hold NaN."""
    rows, columns = x.shape
    flat = torch.full((offset + rows * stride,), float("nan"), dtype=TORCH[type])
    flat[offset:].view(rows, stride)[:, :columns] = torch.from_numpy(np.array(x, np.float32)).to(TORCH[type])
    flat = flat.cuda()
    return flat, flat.data_ptr() + offset * flat.element_size()


class Encoded:
    """Guarded output buffers of codes and scales."""

    def __init__(self, rows, columns, code, block_rows, stride=None, offset=0, scale_pad=0):
        self.rows, self.columns, self.code = rows, columns, code
        self.stride = columns if stride is None else stride
        self.nb, self.nr = -(-columns // 128), -(-rows // block_rows)
        self.scale_stride = self.nr + scale_pad
        self.offset = offset
        self.codes = torch.full((offset + rows * self.stride + 16,), GUARD, dtype=torch.uint8,
                                device="cuda")
        self.scales = torch.full((self.nb * self.scale_stride + 4,), -7.0, device="cuda")

    @property
    def code_ptr(self):
        return self.codes.data_ptr() + self.offset

    def read(self):
        torch.cuda.synchronize()
        flat = self.codes.cpu().numpy()
        body = flat[self.offset:self.offset + self.rows * self.stride].reshape(self.rows, self.stride)
        assert (flat[:self.offset] == GUARD).all() and (flat[-16:] == GUARD).all()
        assert (body[:, self.columns:] == GUARD).all()
        s = self.scales.cpu().numpy()
        assert (s[-4:] == -7.0).all()
        s = s[:-4].reshape(self.nb, self.scale_stride)
        assert (s[:, self.nr:] == -7.0).all()
        return ref.code_values(self.code)[body[:, :self.columns]], s[:, :self.nr].copy()


def run_encode(ws, x, type, code, block_rows, x_stride=None, x_offset=0, stride=None, offset=0,
               scale_pad=0, stream=0):
    rows, columns = x.shape
    x_stride = columns if x_stride is None else x_stride
    keep, ptr = device_matrix(x, type, x_stride, x_offset)
    out = Encoded(rows, columns, code, block_rows, stride, offset, scale_pad)
    ws.encode_scaled(code, type, block_rows, ptr, x_stride, rows, columns, out.code_ptr,
                     out.stride, out.scales.data_ptr(), out.scale_stride, stream)
    got = out.read()
    del keep
    return got


def check_encode(got, x, type, code, block_rows):
    want, scales = ref.encode(rounded(x, type), code, block_rows)
    np.testing.assert_array_equal(got[1], scales)
    np.testing.assert_array_equal(got[0], want)


def values(rows, columns, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((rows, columns)) * np.exp(spread * rng.standard_normal(columns))


SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (2, 4096), (130, 300), (128, 128), (129, 1000),
          (257, 8), (33, 2049)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_encode_equals_the_definition(ws, shape, type, block_rows):
    for code in (ref.E4M3, ref.E5M2):
        x = values(*shape, seed=shape[0] + shape[1])
        check_encode(run_encode(ws, x, type, code, block_rows), x, type, code, block_rows)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("layout", [dict(x_stride=304, stride=304, scale_pad=3),
                                    dict(x_stride=301, x_offset=1, stride=301, offset=1),
                                    dict(x_stride=304, stride=303, offset=5),
                                    dict(x_stride=303, x_offset=3, stride=320, scale_pad=1),
                                    dict(x_stride=300, x_offset=8, stride=308, offset=8)])
def test_encode_strides_and_alignments(ws, type, block_rows, layout):
    x = values(131, 300, seed=5)
    got = run_encode(ws, x, type, ref.E4M3, block_rows, **layout)
    check_encode(got, x, type, ref.E4M3, block_rows)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("code", [ref.E4M3, ref.E5M2])
def test_encode_values_at_the_edges(ws, type, block_rows, code):
    top = {FP32: 3.4028235e38, BF16: 3.3895314e38, FP16: 65504.0}[type]
    tiny = {FP32: 2.0 ** -149, BF16: 2.0 ** -133, FP16: 2.0 ** -24}[type]
    x = np.zeros((9, 512))
    x[1, 0] = top
    x[1, 1] = -top / 2
    x[2, :128] = top
    x[3, 5] = tiny
    x[3, 200] = -tiny
    x[4] = values(1, 512, 1)[0]
    x[4, 3], x[4, 130], x[4, 131] = np.inf, -np.inf, np.nan
    x[5] = np.nan
    x[6] = np.inf
    x[7, :] = np.linspace(-1, 1, 512)
    x[8, 511] = -0.0
    if block_rows == 128:  # one class of value per row group
        x = np.repeat(x, 128, 0)
    check_encode(run_encode(ws, x, type, code, block_rows), x, type, code, block_rows)


def test_encode_ties_go_as_the_division_rounds(ws):
    # every quotient of two small integers: many fall on or beside a tie
    a = np.arange(1, 449, dtype=np.float64)
    x = np.zeros((448, 128))
    for r in range(448):
        x[r] = np.resize(a[:r + 1][::-1], 128)
        x[r, 0] = r + 1
    check_encode(run_encode(ws, x, FP32, ref.E4M3, 1), x, FP32, ref.E4M3, 1)
    check_encode(run_encode(ws, x, BF16, ref.E5M2, 1), x, BF16, ref.E5M2, 1)


def run_norm(ws, x, residual, weight, eps, type, code, x_stride=None, residual_stride=None,
             into=None, stride=None, offset=0, x_offset=0, scale_pad=0):
    """into: None (no stream out), "new", "residual" or "x" (in place)."""
    rows, columns = x.shape
    x_stride = columns if x_stride is None else x_stride
    residual_stride = columns if residual_stride is None else residual_stride
    xk, xp = device_matrix(x, type, x_stride, x_offset)
    rk, rp = (None, 0) if residual is None else device_matrix(residual, type, residual_stride)
    wk, wp = (None, 0) if weight is None else device_matrix(weight[None], type, columns)
    after, ap = None, 0
    if into == "new":
        after = torch.full((rows * residual_stride,), float("nan"), dtype=TORCH[type], device="cuda")
        ap = after.data_ptr()
    elif into == "residual":
        after, ap = rk, rp
    elif into == "x":
        after, ap = xk, xp
    out = Encoded(rows, columns, code, 1, stride, offset, scale_pad)
    ws.rms_norm_scaled(code, type, xp, x_stride, rp, ap, residual_stride, wp, eps, rows, columns,
                       out.code_ptr, out.stride, out.scales.data_ptr(), out.scale_stride)
    got = out.read()
    if after is not None:
        first = x_offset if into == "x" else 0
        after = after[first:].view(rows, residual_stride).double().cpu().numpy()
        assert np.isnan(after[:, columns:]).all()
        after = after[:, :columns]
    return got, after


def check_norm(got, after, x, residual, weight, eps, type, code):
    x, columns = rounded(x, type), x.shape[1]
    residual = None if residual is None else rounded(residual, type)
    weight = None if weight is None else rounded(weight, type)
    h, y = ref.rms_norm(x, residual, weight, eps)
    ref.check_codes(got[0], got[1], y, code, 1, ref.norm_tolerance(columns))
    if after is not None:
        h32 = x if residual is None else x + residual  # FP32, then one rounding
        np.testing.assert_array_equal(after, rounded(h32, type))


@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 127), (5, 129), (7, 1000), (2, 8192),
                                   (130, 300), (4, 16384), (3, 33000), (9, 64), (2, 5001)])
@pytest.mark.parametrize("type", [FP32, BF16, FP16])
def test_norm_against_64_bits(ws, shape, type):
    x, residual = values(*shape, seed=2, spread=0.5), values(*shape, seed=3, spread=0.5)
    weight = 1 + 0.1 * np.random.default_rng(4).standard_normal(shape[1])
    for code, res, w, into in ((ref.E4M3, residual, weight, "new"), (ref.E5M2, None, weight, None),
                               (ref.E4M3, residual, None, "residual"),
                               (ref.E4M3, residual, weight, "x"), (ref.E4M3, None, None, "new"),
                               (ref.E4M3, residual, weight, None)):
        got, after = run_norm(ws, x, res, w, 1e-5, type, code, into=into)
        check_norm(got, after, x, res, w, 1e-5, type, code)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("layout", [dict(x_stride=304, residual_stride=304, stride=304, scale_pad=3),
                                    dict(x_stride=301, x_offset=1, residual_stride=303, stride=301,
                                         offset=1),
                                    dict(x_stride=304, residual_stride=303, stride=303, offset=5),
                                    dict(x_stride=303, x_offset=3, residual_stride=304, stride=320)])
def test_norm_strides_and_alignments(ws, type, layout):
    x, residual = values(11, 300, 5), values(11, 300, 6)
    weight = 1 + 0.1 * np.random.default_rng(4).standard_normal(300)
    got, after = run_norm(ws, x, residual, weight, 1e-6, type, ref.E4M3, into="new", **layout)
    check_norm(got, after, x, residual, weight, 1e-6, type, ref.E4M3)


def test_norm_rows_that_hold_nothing_or_what_is_not_finite(ws):
    x = values(6, 384, 7)
    x[1] = 0
    x[2, 5] = np.inf
    x[3, 300] = np.nan
    x[4] = 1e-30
    x[5, :128] = 0
    got, after = run_norm(ws, x, None, None, 1e-5, FP32, ref.E4M3, into="new")
    check_norm(got, after, x, None, None, 1e-5, FP32, ref.E4M3)
    assert (got[0][1] == 0).all() and np.isnan(got[0][3]).all()
    # eps = 0 on a row of zeros is 0 times infinity
    got, _ = run_norm(ws, x[1:2], None, None, 0.0, FP32, ref.E4M3)
    assert np.isnan(got[0]).all()


def operand(rows, columns, code, block_rows, seed):
    """Random finite codes over the format's range and scales."""
    rng = np.random.default_rng(seed)
    table = ref.code_values(code)
    usable = np.flatnonzero(np.isfinite(table) & (np.abs(table) <= (448 if code == 0 else 64)))
    codes = rng.choice(usable, size=(rows, columns)).astype(np.uint8)
    shape = (-(-columns // 128), -(-rows // block_rows))
    scales = np.exp(rng.standard_normal(shape)).astype(np.float32) * np.float32(2.0 ** -9)
    return codes, scales


def device_codes(codes, stride, offset, filler):
    rows, columns = codes.shape
    flat = torch.full((offset + rows * stride,), filler, dtype=torch.uint8)
    flat[offset:].view(rows, stride)[:, :columns] = torch.from_numpy(codes)
    flat = flat.cuda()
    # what follows the last row's codes is not part of the matrix
    return flat, flat.data_ptr() + offset


def up16(n):
    return -(-n // 16) * 16


def run_gemm(ws, a, a_scales, b, b_scales, a_code, b_code, type, a_stride=None, b_stride=None,
             a_offset=0, b_offset=0, out_stride=None, scale_pad=0, stream=0):
    (m, k), n = a.shape, b.shape[0]
    a_stride = up16(k) if a_stride is None else a_stride
    b_stride = up16(k) if b_stride is None else b_stride
    out_stride = n if out_stride is None else out_stride
    ak, ap = device_codes(a, a_stride, a_offset, 0x7f)  # NaN around the codes
    bk, bp = device_codes(b, b_stride, b_offset, 0x7f)

    def padded(s):
        wide = np.full((s.shape[0], s.shape[1] + scale_pad), np.nan, np.float32)
        wide[:, :s.shape[1]] = s
        return torch.from_numpy(wide).cuda()

    sa, sb = padded(a_scales), padded(b_scales)
    out = torch.full((m * out_stride + 8,), 77.0, dtype=TORCH[type], device="cuda")
    ws.gemm_scaled(a_code, b_code, type, ap, a_stride, sa.data_ptr(), sa.shape[1], bp, b_stride,
                   sb.data_ptr(), sb.shape[1], m, n, k, out.data_ptr(), out_stride, stream)
    torch.cuda.synchronize()
    assert ws.status() == 0
    out = out.double().cpu().numpy()
    assert (out[m * out_stride:] == 77.0).all()
    out = out[:m * out_stride].reshape(m, out_stride)
    assert (out[:, n:] == 77.0).all()
    del ak, bk
    return out[:, :n]


def check_gemm(got, a, a_scales, b, b_scales, a_code, b_code, type):
    want, size = ref.gemm(ref.code_values(a_code)[a], a_scales, ref.code_values(b_code)[b], b_scales)
    bound = ref.gemm_tolerance(a.shape[1]) * size
    # the kernel's FP32 sum lies within the bound and is rounded once: rounding
    # keeps order, so the result lies between the roundings of the two ends
    low, high = rounded(want - bound, type), rounded(want + bound, type)
    assert np.isfinite(got).all()
    assert np.all((low <= got) & (got <= high)), np.max(np.abs(got - want) / (bound + 1e-300))


M = [1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 65, 127, 128, 129, 200, 257]


@pytest.mark.parametrize("m", M)
@pytest.mark.parametrize("nk", [(1, 1), (16, 128), (40, 15), (127, 129), (128, 256), (129, 1000),
                                (300, 1999), (520, 640), (257, 16), (640, 4096)])
def test_gemm_against_64_bits(ws, m, nk):
    n, k = nk
    a, sa = operand(m, k, ref.E4M3, 1, m + k)
    b, sb = operand(n, k, ref.E4M3, 128, n + 2 * k)
    type = (m + n) % 3
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, type)
    check_gemm(got, a, sa, b, sb, ref.E4M3, ref.E4M3, type)


@pytest.mark.parametrize("a_code", [ref.E4M3, ref.E5M2])
@pytest.mark.parametrize("b_code", [ref.E4M3, ref.E5M2])
@pytest.mark.parametrize("m", [1, 12, 48, 150, 300])
@pytest.mark.parametrize("type", [FP32, BF16, FP16])
def test_gemm_codes_and_types(ws, a_code, b_code, m, type):
    a, sa = operand(m, 700, a_code, 1, 1)
    b, sb = operand(330, 700, b_code, 128, 2)
    got = run_gemm(ws, a, sa, b, sb, a_code, b_code, type)
    check_gemm(got, a, sa, b, sb, a_code, b_code, type)


@pytest.mark.parametrize("m", [1, 5, 20, 70, 140])
@pytest.mark.parametrize("layout", [dict(a_stride=500, b_stride=500),
                                    dict(a_stride=512, b_stride=528, out_stride=333, scale_pad=3),
                                    dict(a_offset=1), dict(b_offset=3),
                                    dict(a_offset=16, b_offset=32, out_stride=304),
                                    dict(a_stride=501, b_stride=512)])
def test_gemm_strides_and_alignments(ws, m, layout):
    a, sa = operand(m, 500, ref.E4M3, 1, 3)
    b, sb = operand(300, 500, ref.E4M3, 128, 4)
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, BF16, **layout)
    check_gemm(got, a, sa, b, sb, ref.E4M3, ref.E4M3, BF16)


@pytest.mark.parametrize("size", [(300, 10300, 200), (513, 7700, 1000), (1000, 2600, 129),
                                  (130, 30000, 64), (100, 19000, 130), (20, 9500, 300),
                                  (17, 40000, 16)])
@pytest.mark.parametrize("codes", [(ref.E4M3, ref.E4M3), (ref.E5M2, ref.E4M3)])
@pytest.mark.parametrize("type", [FP32, BF16])
def test_gemm_wide(ws, size, codes, type):
    m, n, k = size
    a, sa = operand(m, k, codes[0], 1, m)
    b, sb = operand(n, k, codes[1], 128, n)
    got = run_gemm(ws, a, sa, b, sb, *codes, type)
    check_gemm(got, a, sa, b, sb, *codes, type)


@pytest.mark.parametrize("size", [(150, 300, 2000), (300, 10300, 2000)])
def test_gemm_wait_that_runs_out(size):
    """A stage whose copies are withheld: NaN, the sticky status, and a context
    that works on."""
    w = _lib.Workspace(0)
    m, n, k = size
    a, sa = operand(m, k, ref.E4M3, 1, 1)
    b, sb = operand(n, k, ref.E4M3, 128, 2)
    w.inject_stall(3, 2_000_000)
    dev = [torch.from_numpy(v).cuda() for v in (a, sa, b, sb)]
    out = torch.zeros(m, n, device="cuda")

    def product():
        w.gemm_scaled(0, 0, FP32, dev[0].data_ptr(), k, dev[1].data_ptr(), sa.shape[1],
                      dev[2].data_ptr(), k, dev[3].data_ptr(), sb.shape[1], m, n, k,
                      out.data_ptr(), n)
        torch.cuda.synchronize()

    product()
    assert w.status() == _lib.STATUS_WAIT_TIMEOUT
    assert torch.isnan(out).any()
    w.inject_stall()
    product()
    assert w.status() == 0
    check_gemm(out.double().cpu().numpy(), a, sa, b, sb, 0, 0, FP32)
    w.close()


@pytest.mark.parametrize("m", [1, 4, 24, 100, 300])
def test_gemm_many_blocks_of_k(ws, m):
    a, sa = operand(m, 20000, ref.E4M3, 1, 3)
    b, sb = operand(70, 20000, ref.E4M3, 128, 4)
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32)
    check_gemm(got, a, sa, b, sb, ref.E4M3, ref.E4M3, FP32)


@pytest.mark.parametrize("m", [3, 40, 150, 300])
def test_gemm_keeps_nan_and_infinity_in_their_rows(ws, m):
    n, k = 300, 400
    a, sa = operand(m, k, ref.E5M2, 1, 3)
    b, sb = operand(n, k, ref.E4M3, 128, 4)
    clean = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E4M3, FP32)
    a[1, 7], b[5, 390] = 0x7f, 0xff  # NaN codes
    b[6, :] = np.where(b[6] & 0x7f == 0, 0x38, b[6])  # no zeros against infinity
    a[2, 3] = 0x7c  # infinity
    got = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E4M3, FP32)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 5]).all()
    assert not np.isfinite(got[2]).any()
    rows, columns = [i for i in range(m) if i not in (1, 2)], [j for j in range(n) if j not in (5, 6)]
    np.testing.assert_array_equal(got[np.ix_(rows, columns)], clean[np.ix_(rows, columns)])


@pytest.mark.parametrize("m", [1, 8, 9, 16])
@pytest.mark.parametrize("k", [8191, 8192, 8193, 8207, 8320, 9000, 20011])
@pytest.mark.parametrize("type", [FP32, FP16])
def test_gemm_few_rows_share_a_long_k(ws, m, k, type):
    n = 37 + k % 100
    a, sa = operand(m, k, ref.E4M3, 1, m)
    b, sb = operand(n, k, ref.E5M2, 128, k)
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E5M2, type)
    check_gemm(got, a, sa, b, sb, ref.E4M3, ref.E5M2, type)
    np.testing.assert_array_equal(run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E5M2, type), got)


@pytest.mark.parametrize("m", [1, 20, 33, 64, 65, 130])
@pytest.mark.parametrize("k", [1, 2, 3, 5, 126, 127, 129, 131, 255, 383, 640])
def test_gemm_rows_on_any_boundary(ws, m, k):
    n, a_code, b_code = 140, (m + k) % 2, (m // 2 + k) % 2
    a, sa = operand(m, k, a_code, 1, m)
    b, sb = operand(n, k, b_code, 128, k)
    # rows on every offset from 4 bytes on both sides; NaN codes around the rows
    for layout in (dict(a_stride=k + 1 - k % 2, b_stride=k + 3 - k % 2, a_offset=1),
                   dict(a_stride=up16(k) + 2, b_stride=up16(k) + 4, b_offset=3),
                   dict(a_stride=up16(k), b_stride=up16(k) + 7)):
        got = run_gemm(ws, a, sa, b, sb, a_code, b_code, FP32, **layout)
        check_gemm(got, a, sa, b, sb, a_code, b_code, FP32)


@pytest.mark.parametrize("m", [10, 70])
def test_gemm_keeps_nan_and_infinity_in_their_rows_on_any_boundary(ws, m):
    n, k = 150, 403
    a, sa = operand(m, k, ref.E5M2, 1, 3)
    b, sb = operand(n, k, ref.E4M3, 128, 4)
    layout = dict(a_stride=k, b_stride=k, a_offset=1)
    clean = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E4M3, FP32, **layout)
    a[1, 402], b[5, 0] = 0x7f, 0xff  # NaN codes
    b[b & 0x7f == 0] = 0x38  # no zeros against infinity
    clean_again = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E4M3, FP32, **layout)
    a[2, 3] = 0x7c  # infinity
    got = run_gemm(ws, a, sa, b, sb, ref.E5M2, ref.E4M3, FP32, **layout)
    assert np.isfinite(clean).all()
    assert np.isnan(got[1]).all() and np.isnan(got[:, 5]).all()
    assert not np.isfinite(got[2]).any()
    rows, columns = [i for i in range(m) if i not in (1, 2)], [j for j in range(n) if j != 5]
    np.testing.assert_array_equal(got[np.ix_(rows, columns)], clean_again[np.ix_(rows, columns)])
    assert np.isfinite(got[np.ix_(rows, columns)]).all()


@pytest.mark.parametrize("m", [2, 30, 200])
def test_gemm_zero_rows_and_repeats(ws, m):
    a, sa = operand(m, 1024, ref.E4M3, 1, 3)
    b, sb = operand(512, 1024, ref.E4M3, 128, 4)
    a[m - 1] = 0
    b[100] = 0x80  # minus zero
    first = run_gemm(ws, a, sa, b, sb, 0, 0, BF16)
    assert (first[m - 1] == 0).all() and (first[:, 100] == 0).all()
    for _ in range(3):  # sums are joined in a fixed order
        np.testing.assert_array_equal(run_gemm(ws, a, sa, b, sb, 0, 0, BF16), first)


def test_gemm_degenerate_sizes(ws):
    out = torch.full((3, 5), 7.0, device="cuda")
    ws.gemm_scaled(0, 0, FP32, 0, 0, 0, 0, 0, 0, 0, 0, 3, 5, 0, out.data_ptr(), 5)
    torch.cuda.synchronize()
    assert (out == 0).all()
    ws.gemm_scaled(0, 0, FP32, 0, 0, 0, 0, 0, 0, 0, 0, 0, 5, 9, 0, 5)
    ws.gemm_scaled(0, 0, FP32, 0, 0, 0, 0, 0, 0, 0, 0, 3, 0, 9, 0, 5)
    ws.encode_scaled(0, FP32, 1, 0, 0, 0, 5, 0, 0, 0, 0)
    ws.encode_scaled(0, FP32, 128, 0, 0, 5, 0, 0, 0, 0, 0)
    ws.rms_norm_scaled(0, FP32, 0, 0, 0, 0, 0, 0, 1e-5, 0, 8, 0, 0, 0, 0)


@pytest.mark.parametrize("m", [1, 150])
def test_gemm_offsets_past_32_bits(ws, m):
    # rows 2^31 bytes apart: the last starts beyond 2^32
    n, k, stride = 4, 300, (1 << 31) + 16
    a, sa = operand(m, k, ref.E4M3, 1, 3)
    b, sb = operand(n, k, ref.E4M3, 128, 4)
    flat = torch.empty(3 * stride + 304, dtype=torch.uint8, device="cuda")
    for r in range(n):
        flat[r * stride:r * stride + k] = torch.from_numpy(b[r]).cuda()
    ak, ap = device_codes(a, 304, 0, 0x7f)
    out = torch.zeros(m, n, device="cuda")
    s0, s1 = torch.from_numpy(sa).cuda(), torch.from_numpy(sb).cuda()
    ws.gemm_scaled(0, 0, FP32, ap, 304, s0.data_ptr(), m, flat.data_ptr(), stride, s1.data_ptr(),
                   1, m, n, k, out.data_ptr(), n)
    torch.cuda.synchronize()
    check_gemm(out.double().cpu().numpy(), a, sa, b, sb, 0, 0, FP32)
    # and out rows 2^31 elements apart
    ws.gemm_scaled(0, 0, BF16, ap, 304, s0.data_ptr(), m, flat.data_ptr(), stride, s1.data_ptr(),
                   1, min(m, 2), n, k, flat.data_ptr() + 512, 1 << 30)
    torch.cuda.synchronize()
    for r in range(min(m, 2)):
        at = 512 + (r << 31)
        got = flat[at:at + 2 * n].view(torch.bfloat16).double().cpu().numpy()[None]
        check_gemm(got, a[r:r + 1], sa[:, r:r + 1], b, sb, 0, 0, BF16)
    assert ws.status() == 0
    del ak


def test_encode_and_norm_offsets_past_32_bits(ws):
    rows, columns, stride = 3, 200, (1 << 31) + 8
    x = values(rows, columns, 9)
    flat = torch.empty(2 * stride + columns, dtype=torch.bfloat16, device="cuda")
    for r in range(rows):
        flat[r * stride:r * stride + columns] = torch.from_numpy(x[r]).bfloat16().cuda()
    out = Encoded(rows, columns, 0, 1)
    ws.encode_scaled(0, BF16, 1, flat.data_ptr(), stride, rows, columns, out.code_ptr, columns,
                     out.scales.data_ptr(), rows)
    check_encode(out.read(), x, BF16, 0, 1)
    out = Encoded(rows, columns, 0, 1)
    ws.rms_norm_scaled(0, BF16, flat.data_ptr(), stride, 0, 0, 0, 0, 1e-5, rows, columns,
                       out.code_ptr, columns, out.scales.data_ptr(), rows)
    check_norm(out.read(), None, x, None, None, 1e-5, BF16, 0)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_operators_follow_their_stream_and_replay_in_a_graph(ws, m):
    """norm -> product on a stream of their own, then captured and replayed on
    new inputs."""
    n, k = 256, 512
    weight = values(1, k, 1)[0] * 0 + 1.5
    b, sb = operand(n, k, 0, 128, 2)
    bd, sbd = torch.from_numpy(b).cuda(), torch.from_numpy(sb).cuda()
    wd = torch.from_numpy(weight).bfloat16().cuda()
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    codes = torch.empty(m, k, dtype=torch.uint8, device="cuda")
    scales = torch.empty(k // 128, m, device="cuda")
    out = torch.empty(m, n, device="cuda")

    def step(stream):
        ws.rms_norm_scaled(0, BF16, x.data_ptr(), k, 0, 0, 0, wd.data_ptr(), 1e-5, m, k,
                           codes.data_ptr(), k, scales.data_ptr(), m, stream)
        ws.gemm_scaled(0, 0, FP32, codes.data_ptr(), k, scales.data_ptr(), m, bd.data_ptr(), k,
                       sbd.data_ptr(), sbd.shape[1], m, n, k, out.data_ptr(), n, stream)

    def check():
        c, s = codes.cpu().numpy(), scales.cpu().numpy()
        h, y = ref.rms_norm(x.double().cpu().numpy(), None, rounded(weight, BF16), 1e-5)
        ref.check_codes(ref.code_values(0)[c], s, y, 0, 1, ref.norm_tolerance(k))
        check_gemm(out.double().cpu().numpy(), c, s, b, sb, 0, 0, FP32)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for seed in range(20):
            x.copy_(torch.from_numpy(values(m, k, seed)).pin_memory(), non_blocking=True)
            step(stream.cuda_stream)
    stream.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in (30, 31):
        x.copy_(torch.from_numpy(values(m, k, seed)))
        graph.replay()
        torch.cuda.synchronize()
        check()


def test_refusals(ws):
    buf = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    p = (buf.data_ptr() + 255) // 256 * 256

    def refused(status, text, call, *args):
        with pytest.raises(_lib.AutError) as info:
            call(*args)
        assert info.value.status == status and text in str(info.value), info.value

    bad, large = _lib.AUT_ERR_INVALID_ARGUMENT, _lib.AUT_ERR_TOO_LARGE
    enc, norm, gemm = ws.encode_scaled, ws.rms_norm_scaled, ws.gemm_scaled
    refused(bad, "code", enc, 2, 0, 1, p, 8, 2, 8, p, 8, p, 2)
    refused(bad, "type", enc, 0, 3, 1, p, 8, 2, 8, p, 8, p, 2)
    refused(bad, "block_rows", enc, 0, 0, 64, p, 8, 2, 8, p, 8, p, 2)
    refused(bad, "values is NULL", enc, 0, 0, 1, 0, 8, 2, 8, p, 8, p, 2)
    refused(bad, "codes is NULL", enc, 0, 0, 1, p, 8, 2, 8, 0, 8, p, 2)
    refused(bad, "scales is NULL", enc, 0, 0, 1, p, 8, 2, 8, p, 8, 0, 2)
    refused(bad, "values: stride", enc, 0, 0, 1, p, 7, 2, 8, p, 8, p, 2)
    refused(bad, "codes: stride", enc, 0, 0, 1, p, 8, 2, 8, p, 7, p, 2)
    refused(bad, "scales: stride", enc, 0, 0, 1, p, 200, 2, 200, p, 200, p, 1)
    refused(bad, "aligned", enc, 0, 0, 1, p + 2, 8, 2, 8, p, 8, p, 2)
    refused(bad, "aligned", enc, 0, 1, 1, p + 1, 8, 2, 8, p, 8, p, 2)
    refused(bad, "aligned", enc, 0, 0, 1, p, 8, 2, 8, p, 8, p + 2, 2)
    refused(large, "2^31", enc, 0, 0, 1, p, 1 << 40, 1 << 31, 8, p, 8, p, 1 << 31)
    refused(large, "2^53", enc, 0, 0, 1, p, 1 << 60, 3, 8, p, 8, p, 3)
    refused(bad, "eps", norm, 0, 0, p, 8, 0, 0, 0, 0, -1.0, 2, 8, p, 8, p, 2)
    refused(bad, "eps", norm, 0, 0, p, 8, 0, 0, 0, 0, float("nan"), 2, 8, p, 8, p, 2)
    refused(bad, "x is NULL", norm, 0, 0, 0, 8, 0, 0, 0, 0, 0.0, 2, 8, p, 8, p, 2)
    refused(bad, "residual: stride", norm, 0, 0, p, 8, p, 0, 7, 0, 0.0, 2, 8, p, 8, p, 2)
    refused(bad, "residual_out: stride", norm, 0, 0, p, 8, 0, p, 7, 0, 0.0, 2, 8, p, 8, p, 2)
    refused(bad, "another stride", norm, 0, 0, p, 8, 0, p, 9, 0, 0.0, 2, 8, p, 8, p, 2)
    refused(bad, "weight", norm, 0, 0, p, 8, 0, 0, 0, p + 2, 0.0, 2, 8, p, 8, p, 2)
    good = [0, 0, 0, p, 256, p, 2, p, 256, p, 2, 2, 200, 256, p, 200]
    for at, value, status, text in ((0, 5, bad, "code"), (1, -1, bad, "code"), (2, 9, bad, "type"),
                                    (3, 0, bad, "a is NULL"), (4, 255, bad, "a: stride"),
                                    (5, 0, bad, "a_scales is NULL"), (6, 1, bad, "a_scales: stride"),
                                    (7, 0, bad, "b is NULL"), (8, 10, bad, "b: stride"),
                                    (9, p + 1, bad, "b_scales"), (10, 1, bad, "b_scales: stride"),
                                    (13, 1 << 31, large, "2^31"), (14, 0, bad, "out is NULL"),
                                    (14, p + 2, bad, "out is not aligned"),
                                    (15, 199, bad, "out: stride"), (4, 1 << 62, large, "2^53")):
        args = list(good)
        args[at] = value
        refused(status, text, gemm, *args)
    assert (buf == 0).all() and ws.status() == 0


@pytest.mark.parametrize("tokens", [1, 12, 150])
def test_feed_forward_example(ws, tokens):
    """The example's block against itself in 64 bits from the decoded weights:
    what is left is the encoding of the activations and of the output."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "examples"))
    import scaled_feed_forward as example
    g = torch.Generator(device="cuda").manual_seed(tokens)
    width, inner = 512, 768

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    gain, x, stream = 1 + normal(width, scale=0.1), normal(tokens, width), normal(tokens, width)
    up, down = normal(2 * inner, width, scale=width ** -0.5), normal(width, inner, scale=inner ** -0.5)
    block = example.FeedForward(ws, gain, up, down)
    before = stream.clone()
    got = block(x, stream)
    torch.testing.assert_close(stream, (x.float() + before.float()).bfloat16(), rtol=0, atol=0)
    want, _ = example.reference(gain, block.up.decoded(), block.down.decoded(), x, before)
    # codes round within 2^-4 of a value, two encodings one behind the other,
    # each error spread over the sums: far below half of 2^-4 in the norm
    assert (got.float() - want).norm() <= 2 ** -4 * want.norm()


def test_tensor_calls(ws):
    from accessor_universal_test_b200 import scaled
    x = torch.randn(70, 300, device="cuda")
    a = scaled.encode(ws, x)
    b = scaled.encode(ws, torch.randn(200, 300, device="cuda"), block_rows=128)
    assert (a.decoded() - x).abs().max() <= x.abs().max() * 2 ** -4
    out = scaled.matmul(ws, a, b, dtype=torch.float32)
    torch.testing.assert_close(out, a.decoded() @ b.decoded().t(), rtol=1e-4, atol=1e-3)
    same = torch.empty_like(out)
    assert scaled.matmul(ws, a, b, out=same) is same and torch.equal(same, out)
    again = scaled.encode(ws, x, out=a)
    assert again is a
    n, s = scaled.rms_norm(ws, x)
    assert s is x and n.codes.shape == (70, 300)
    for bad in (lambda: scaled.encode(ws, x.t()), lambda: scaled.encode(ws, x.double()),
                lambda: scaled.encode(ws, x, out=b), lambda: scaled.rms_norm(ws, x, x[0, :5]),
                lambda: scaled.rms_norm(ws, x, residual=x.bfloat16()),
                lambda: scaled.matmul(ws, a, b, out=out[:, :5]),
                lambda: scaled.matmul(ws, a, b, dtype=torch.float64)):
        with pytest.raises(ValueError):
            bad()
