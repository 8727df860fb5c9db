"""The loops of the block-scaled operators past their first turn: more rows and tiles
than run at one time, and rows that leave 16-byte boundaries one operand at a time."""
import numpy as np
import pytest

import scaled_ref as ref
from test_gpu_scaled import (BF16, FP16, FP32, check_encode, check_gemm, check_norm, operand,
                             run_encode, run_gemm, run_norm, values)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("shape", [(20000, 264), (3000, 4096), (20000, 263), (2999, 4099),
                                   (40003, 8)])
def test_encode_rows_over_several_turns(ws, shape, type):
    x = values(*shape, seed=shape[0])
    x[-1, 3], x[shape[0] // 2, 5], x[7, 7] = np.inf, -np.inf, np.nan
    check_encode(run_encode(ws, x, type, ref.E4M3, 1), x, type, ref.E4M3, 1)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("shape", [(2100, 2500), (4200, 1999), (1153, 7000)])
def test_encode_tiles_over_several_turns(ws, shape, type):
    """More than two tiles to a block, with infinities in early and late ones."""
    x = values(*shape, seed=shape[1])
    x[-1, -1], x[shape[0] // 2, 900], x[3, 3], x[130, 200] = np.inf, -np.inf, np.inf, np.nan
    x[1100:1120, 300:700] = np.inf
    check_encode(run_encode(ws, x, type, ref.E5M2, 128), x, type, ref.E5M2, 128)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("shape", [(5000, 1000), (1500, 5001), (9001, 200), (1300, 6000),
                                   (900, 9000), (700, 16384), (300, 16392), (200, 20001)])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_norm_over_several_turns(ws, shape, type, into):
    """The next row is read before this one's sum goes back in place of an operand."""
    x, residual = values(*shape, seed=2, spread=0.5), values(*shape, seed=3, spread=0.5)
    weight = 1 + 0.1 * np.random.default_rng(4).standard_normal(shape[1])
    got, after = run_norm(ws, x, residual, weight, 1e-5, type, ref.E4M3, into=into)
    check_norm(got, after, x, residual, weight, 1e-5, type, ref.E4M3)


OFF_BY_ONE = [dict(x_offset=1), dict(x_stride=305), dict(offset=1), dict(stride=305),
              dict(offset=4), dict(stride=308), dict(x_offset=4), dict(x_stride=308),
              dict(x_offset=2, offset=2), dict()]


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("layout", OFF_BY_ONE)
def test_encode_leaves_its_boundaries_one_at_a_time(ws, type, block_rows, layout):
    """304 columns: only the pointer or the stride named stands off them."""
    x = values(131, 304, seed=5)
    layout = dict(x_stride=304, stride=304) | layout
    got = run_encode(ws, x, type, ref.E4M3, block_rows, **layout)
    check_encode(got, x, type, ref.E4M3, block_rows)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("columns", [304, 2048, 6000])
@pytest.mark.parametrize("layout", [dict(x_offset=1), dict(x_stride=1), dict(residual_stride=1),
                                    dict(residual_stride=4), dict(offset=1), dict(stride=1),
                                    dict(offset=4), dict(x_offset=4), dict(x_offset=8), dict()])
def test_norm_leaves_its_boundaries_one_at_a_time(ws, type, columns, layout):
    """Strides are the columns plus what stands here."""
    x, residual = values(11, columns, 5), values(11, columns, 6)
    weight = 1 + 0.1 * np.random.default_rng(4).standard_normal(columns)
    layout = dict(layout)
    for name in ("x_stride", "residual_stride", "stride"):
        layout[name] = columns + layout.get(name, 0)
    got, after = run_norm(ws, x, residual, weight, 1e-6, type, ref.E4M3, into="new", **layout)
    check_norm(got, after, x, residual, weight, 1e-6, type, ref.E4M3)


@pytest.mark.parametrize("type", [FP32, BF16, FP16])
@pytest.mark.parametrize("which", ["weight", "residual", "residual_out"])
def test_norm_with_one_pointer_off_its_boundary(ws, type, which):
    import torch
    from test_gpu_scaled import TORCH, Encoded, device_matrix
    rows, columns = 11, 304
    x, residual = values(rows, columns, 5), values(rows, columns, 6)
    weight = 1 + 0.1 * np.random.default_rng(4).standard_normal(columns)
    off = lambda name: int(which == name)  # noqa: E731
    xk, xp = device_matrix(x, type, columns)
    rk, rp = device_matrix(residual, type, columns, off("residual"))
    wk, wp = device_matrix(weight[None], type, columns, off("weight"))
    after = torch.full((rows * columns + 2,), float("nan"), dtype=TORCH[type], device="cuda")
    at = off("residual_out")
    out = Encoded(rows, columns, ref.E4M3, 1)
    ws.rms_norm_scaled(ref.E4M3, type, xp, columns, rp, after.data_ptr() + at * after.element_size(),
                       columns, wp, 1e-6, rows, columns, out.code_ptr, out.stride,
                       out.scales.data_ptr(), out.scale_stride)
    got = out.read()
    after = after.double().cpu().numpy()
    assert np.isnan(after[:at]).all() and np.isnan(after[at + rows * columns:]).all()
    check_norm(got, after[at:at + rows * columns].reshape(rows, columns), x, residual, weight, 1e-6,
               type, ref.E4M3)
    del xk, rk, wk


# tiles of 256 columns (rows of the result on 16 bytes, and not), 128 and 64: several
# tiles to a block and more blocks of k than the ring holds
@pytest.mark.parametrize("size", [(2000, 4000, 1000), (2000, 4001, 1000), (600, 9400, 1100),
                                  (1157, 1851, 850), (2000, 4000, 200)])
@pytest.mark.parametrize("type", [FP32, BF16])
def test_products_of_several_tiles_to_a_block(ws, size, type):
    m, n, k = size
    a, sa = operand(m, k, ref.E4M3, 1, m)
    b, sb = operand(n, k, ref.E5M2, 128, n)
    a[m // 2:m // 2 + 40] = 0  # rows of zeros, as aut_encode_scaled leaves them
    sa[:, m // 2:m // 2 + 40] = 2.0 ** -126
    got = run_gemm(ws, a, sa, b, sb, ref.E4M3, ref.E5M2, type)
    check_gemm(got, a, sa, b, sb, ref.E4M3, ref.E5M2, type)
