"""The bounded waits of the product over tiles: what a block leaves behind where one
runs out, and bounds that are too short to mean a fault."""
import numpy as np
import pytest
import torch

import scaled_ref as ref
from accessor_universal_test_b200 import _lib
from gpu_util import TOL, device_pair, gpu_dot, normalized_error, oracle_dot
from test_gpu_scaled import FP32, check_gemm, operand

pytestmark = pytest.mark.gpu

OFF = 2 ** 64 - 1
# tiles of 32 columns (cut and uncut), 64 (cut and uncut), 128, and 256 (rows of the
# result on 16 bytes, and not)
SIZES = [(64, 1024, 5120), (33, 520, 640), (129, 700, 3000), (150, 3000, 2000), (300, 10300, 2000),
         (300, 6500, 1999), (300, 6501, 1999)]


class Product:
    """A product of operands on the device."""

    def __init__(self, w, m, n, k):
        self.w, self.size = w, (m, n, k)
        a, self.sa = operand(m, k, ref.E4M3, 1, 1)
        b, self.sb = operand(n, k, ref.E4M3, 128, 2)
        self.a, self.b = a, b
        stride = -(-k // 16) * 16
        self.dev = [torch.zeros(x.shape[0], stride, dtype=torch.uint8, device="cuda") for x in (a, b)]
        for to, x in zip(self.dev, (a, b)):
            to[:, :k] = torch.from_numpy(x).cuda()
        self.scales = [torch.from_numpy(s).cuda() for s in (self.sa, self.sb)]

    def __call__(self):
        (m, n, k), (a, b), (sa, sb) = self.size, self.dev, self.scales
        out = torch.zeros(m, n, device="cuda")
        self.w.gemm_scaled(0, 0, FP32, a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0),
                           b.data_ptr(), b.stride(0), sb.data_ptr(), sb.stride(0), m, n, k,
                           out.data_ptr(), n)
        torch.cuda.synchronize()
        return out.double().cpu().numpy()

    def check(self, got):
        check_gemm(got, self.a, self.sa, self.b, self.sb, 0, 0, FP32)


@pytest.mark.parametrize("size", SIZES)
def test_a_bound_of_one_cycle_is_no_fault(size):
    """Bounds shorter than a copy takes count as the shortest one."""
    w = _lib.Workspace(0)
    product = Product(w, *size)
    w.inject_stall(OFF, 1)
    product.check(product())
    assert w.status() == 0
    w.close()


def test_a_bound_of_one_cycle_is_no_fault_of_a_dot(ws, orc):
    x, y = device_pair(ws, "e8m0", _lib.DENSE, 1 << 20)
    ws.inject_stall(OFF, 1)
    try:
        got = gpu_dot(ws, "e8m0", _lib.DENSE, 0, x, y, 1 << 20, strategy=_lib.STRATEGY_TMA)
        assert ws.status() == 0
    finally:
        ws.inject_stall()
    dot, size = oracle_dot(orc, "e8m0", 1 << 20)
    assert normalized_error(got, dot, size) <= TOL[0]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("block", [0, 3])
def test_what_a_block_had_to_write_is_nan(size, block):
    """Every thread block misses one load of its first tile, so nothing that it or
    the blocks it joins with write is a number.  (Of more tiles to a block, the
    later ones too.)"""
    w = _lib.Workspace(0)
    product = Product(w, *size)
    w.inject_stall(block, 1)
    got = product()
    assert w.status() == _lib.STATUS_WAIT_TIMEOUT
    assert np.isnan(got).all()
    w.inject_stall()
    product.check(product())
    assert w.status() == 0
    w.close()
