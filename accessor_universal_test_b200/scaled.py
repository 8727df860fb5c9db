"""Block-scaled 8-bit matrices on torch tensors (torch supplies the memory,
libautdot does the work).

A ``Scaled`` holds the codes of a matrix and its scales.  Weights are encoded
once by blocks of 128 x 128, activations by rows of 128 columns, straight from
the norm that makes them or by ``encode``::

    w = scaled.encode(ws, weight, block_rows=128)            # once
    a, stream = scaled.rms_norm(ws, x, gain, residual=stream)
    y = scaled.matmul(ws, a, w)                              # x.dtype out

Every call runs on torch's current stream of the tensors' device.  None of them
is differentiated: where gradients are recorded, tensors that require one are
refused.  What a call writes in place counts as changed for torch, so a backward
pass that needs the old values says so.
"""
from __future__ import annotations

import torch

from . import _lib

TYPES = {torch.float32: _lib.TYPE_FP32, torch.bfloat16: _lib.TYPE_BF16,
         torch.float16: _lib.TYPE_FP16}


class Scaled:
    """Codes [rows, columns] (uint8, rows a whole number of 16-byte lines apart)
    and scales [ceil(columns / 128), ceil(rows / block_rows)] of a matrix."""

    def __init__(self, rows: int, columns: int, code: int = _lib.FP8_E4M3, block_rows: int = 1,
                 device=None):
        if block_rows not in (1, _lib.SCALE_BLOCK):
            raise ValueError("block_rows must be 1 or 128")
        if code not in (_lib.FP8_E4M3, _lib.FP8_E5M2):
            raise ValueError("code must be FP8_E4M3 or FP8_E5M2")
        stride = -(-columns // 16) * 16
        self.storage = torch.empty(rows, stride, dtype=torch.uint8, device=device)
        self.codes = self.storage[:, :columns]
        self.scales = torch.empty(-(-columns // _lib.SCALE_BLOCK), -(-rows // block_rows),
                                  dtype=torch.float32, device=device)
        self.rows, self.columns, self.code, self.block_rows = rows, columns, code, block_rows

    def decoded(self) -> torch.Tensor:
        """The values in FP32 (a check's form, not a fast one)."""
        kind = torch.float8_e4m3fn if self.code == _lib.FP8_E4M3 else torch.float8_e5m2
        scales = self.scales.t().repeat_interleave(self.block_rows, 0)[:self.rows]
        scales = scales.repeat_interleave(_lib.SCALE_BLOCK, 1)[:, :self.columns]
        return self.codes.contiguous().view(kind).float() * scales


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _written(*tensors: torch.Tensor) -> None:
    """Tells torch of tensors that a call has written through their pointers."""
    torch.autograd.graph.increment_version(tensors)


def _check(name: str, t: torch.Tensor, ws: _lib.Workspace, shape=None, dtype=None) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which these calls do not make "
                         "(detach it, or call under torch.no_grad())")
    if t.device != torch.device("cuda", ws.device):
        raise ValueError(f"{name} is on {t.device}, the workspace on cuda:{ws.device}")
    if t.dtype not in TYPES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} has type {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, wanted {tuple(shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} is not contiguous along its last dimension")


def _out(out: Scaled | None, ws: _lib.Workspace, rows: int, columns: int, code: int,
         block_rows: int) -> Scaled:
    if out is None:
        return Scaled(rows, columns, code, block_rows, torch.device("cuda", ws.device))
    if (out.rows, out.columns, out.code, out.block_rows) != (rows, columns, code, block_rows):
        raise ValueError("out has other sizes, code or block_rows")
    if out.codes.device != torch.device("cuda", ws.device):
        raise ValueError(f"out is on {out.codes.device}, the workspace on cuda:{ws.device}")
    return out


def encode(ws: _lib.Workspace, values: torch.Tensor, code: int = _lib.FP8_E4M3,
           block_rows: int = 1, out: Scaled | None = None) -> Scaled:
    """values [rows, columns] (FP32, BF16 or FP16) as block-scaled codes."""
    if values.dim() != 2:
        raise ValueError("values must have two dimensions")
    _check("values", values, ws)
    rows, columns = values.shape
    out = _out(out, ws, rows, columns, code, block_rows)
    ws.encode_scaled(code, TYPES[values.dtype], block_rows, values.data_ptr(), values.stride(0),
                     rows, columns, out.storage.data_ptr(), out.storage.stride(0),
                     out.scales.data_ptr(), out.scales.stride(0), _stream(values))
    _written(out.storage, out.scales)
    return out


def rms_norm(ws: _lib.Workspace, x: torch.Tensor, weight: torch.Tensor | None = None,
             eps: float = 1e-5, residual: torch.Tensor | None = None, code: int = _lib.FP8_E4M3,
             out: Scaled | None = None) -> tuple[Scaled, torch.Tensor]:
    """(x + residual) / rms * weight encoded by rows, and x + residual in the
    type of x: written into residual, or x itself where there is none."""
    if x.dim() != 2:
        raise ValueError("x must have two dimensions")
    _check("x", x, ws)
    rows, columns = x.shape
    if residual is not None:
        _check("residual", residual, ws, x.shape, x.dtype)
    if weight is not None:
        _check("weight", weight, ws, (columns,), x.dtype)
    out = _out(out, ws, rows, columns, code, 1)
    at = 0 if residual is None else residual.data_ptr()
    ws.rms_norm_scaled(code, TYPES[x.dtype], x.data_ptr(), x.stride(0), at, at,
                       0 if residual is None else residual.stride(0),
                       0 if weight is None else weight.data_ptr(), eps, rows, columns,
                       out.storage.data_ptr(), out.storage.stride(0), out.scales.data_ptr(),
                       out.scales.stride(0), _stream(x))
    _written(out.storage, out.scales)
    if residual is None:
        return out, x
    _written(residual)
    return out, residual


def matmul(ws: _lib.Workspace, a: Scaled, b: Scaled, dtype: torch.dtype = torch.bfloat16,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """a [m, k] (scales by rows) times b [n, k] transposed (scales by 128 rows)."""
    if a.block_rows != 1 or b.block_rows != _lib.SCALE_BLOCK:
        raise ValueError("a takes scales by rows, b by blocks of 128 rows")
    if a.columns != b.columns:
        raise ValueError(f"a has {a.columns} columns, b {b.columns}")
    for name, t in (("a", a.codes), ("b", b.codes)):
        if t.device != torch.device("cuda", ws.device):
            raise ValueError(f"{name} is on {t.device}, the workspace on cuda:{ws.device}")
    if out is None:
        if dtype not in TYPES:
            raise ValueError(f"no product of type {dtype}")
        out = torch.empty(a.rows, b.rows, dtype=dtype, device=a.codes.device)
    _check("out", out, ws, (a.rows, b.rows))
    ws.gemm_scaled(a.code, b.code, TYPES[out.dtype], a.storage.data_ptr(), a.storage.stride(0),
                   a.scales.data_ptr(), a.scales.stride(0), b.storage.data_ptr(),
                   b.storage.stride(0), b.scales.data_ptr(), b.scales.stride(0), a.rows, b.rows,
                   a.columns, out.data_ptr(), out.stride(0), _stream(out))
    _written(out)
    return out
