"""Microscaled 4-bit floating point (OCP MXFP4): quantisation, and products with operands held in it.

A weight in MXFP4 takes 17/32 of a byte an element.  ``mxfp4_linear`` multiplies bf16 activations by it
(a frozen base weight: the reference's profiles keep theirs in another 4-bit format through another
library) and ``mxfp4_linear_backward`` is the gradient for the activations; ``mxfp4_gemm`` multiplies two
MXFP4 operands on the scaled matrix instructions.  ``autograd.mxfp4_linear`` and
``autograd.lora_linear_compressed`` (an ``MXFP4Tensor`` as its base weight) call them.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from ._lib import LrqMxfp4, call, call_raw, check
from .api import _on, _p, _require_device, _stream
from .norm import _dtype, _rows

__all__ = ["MXFP4Tensor", "mxfp4_quantize", "mxfp4_dequantize", "mxfp4_gemm", "mxfp4_linear", "mxfp4_linear_backward"]


@dataclass(eq=False)
class MXFP4Tensor:
    """A tensor [..., cols] in MXFP4; rows are its leading dimensions flattened.

    ``codes`` uint8 [rows, >= 64 ceil(cols / 128)]: e2m1 elements, the even column in a byte's low nibble.
    ``scales`` uint8 [rows, >= 4 ceil(cols / 128)]: one E8M0 exponent for 32 columns.  Columns past ``cols``
    have code 0 and a scale below 255."""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> "MXFP4Tensor":
        return MXFP4Tensor(self.codes.to(device), self.scales.to(device), self.shape)

    def descriptor(self) -> LrqMxfp4:
        c, s, shape = self.codes, self.scales, self.shape
        _require_device(c, s)
        cols = shape[-1] if len(shape) else 0
        if cols <= 0:
            raise ValueError("an MXFP4 tensor needs rows of at least one element")
        rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
        steps = (cols + 127) // 128
        if c.dim() == 2 and s.dim() == 2 and c.dtype is torch.uint8 and s.dtype is torch.uint8 and c.device == s.device:
            (cr, cw), (sr, sw), (ldc, c1), (lds, s1) = c.shape, s.shape, c.stride(), s.stride()
            if cr == rows and sr == rows and cw >= 64 * steps and sw >= 4 * steps and c1 == 1 and s1 == 1:
                if rows <= 1:  # the stride of a single row means nothing
                    ldc, lds = 64 * steps, 4 * steps
                return LrqMxfp4(c.data_ptr(), ldc, s.data_ptr(), lds, rows, cols)
        raise ValueError(f"codes and scales must be uint8 [{rows}, >= {64 * steps}] and [{rows}, >= {4 * steps}] with unit "
                         f"inner stride on one device, got {c.dtype} {tuple(c.shape)} on {c.device} and {s.dtype} "
                         f"{tuple(s.shape)} on {s.device}")


def mxfp4_quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x[..., n] (bf16, fp16 or fp32) in MXFP4: per 32 columns of a row the scale 2^(floor(log2 max|x|) - 2),
    elements rounded to the nearest code (ties to the even one) and saturated.  A block with an infinity
    or a NaN becomes NaN."""
    _require_device(x)
    dt = _dtype(x, "x")
    x2, rows, n, ldx = _rows(x, "x")
    steps = (n + 127) // 128
    codes = x.new_empty((rows, 64 * steps), dtype=torch.uint8)
    scales = x.new_empty((rows, 4 * steps), dtype=torch.uint8)
    t = LrqMxfp4(codes.data_ptr(), 64 * steps, scales.data_ptr(), 4 * steps, rows, n)
    with _on(x.device):
        call("lrq_mxfp4_quantize", _p(x2), ldx, dt, ctypes.byref(t), _stream(x.device))
    return MXFP4Tensor(codes, scales, tuple(x.shape))


def mxfp4_dequantize(q: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of q (exact in bf16 and fp32)."""
    t = q.descriptor()
    out = q.codes.new_empty(q.shape, dtype=dtype)
    with _on(q.device):
        call("lrq_mxfp4_dequantize", ctypes.byref(t), _p(out), q.cols, _dtype(out, "the output"), _stream(q.device))
    return out


def _out_fp32(out_dtype) -> int:
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("out_dtype must be float32 or bfloat16")
    return 1 if out_dtype == torch.float32 else 0


def _matrix(w: MXFP4Tensor, device: torch.device) -> LrqMxfp4:
    if len(w.shape) != 2:
        raise ValueError(f"an MXFP4 weight must be a matrix, got {tuple(w.shape)}")
    if w.device != device:
        raise ValueError(f"the weight is on {w.device}, the operand on {device}")
    return w.descriptor()


def mxfp4_gemm(a: MXFP4Tensor, b: MXFP4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a @ b^T for a [..., K] and b [N, K], both MXFP4: [..., N], fp32 accumulate."""
    f32 = _out_fp32(out_dtype)
    tb = _matrix(b, a.device)
    ta = a.descriptor()
    if a.cols != b.cols:
        raise ValueError(f"operands have {a.cols} and {b.cols} columns")
    out = a.codes.new_empty((ta.rows, tb.rows) if len(a.shape) == 2 else tuple(a.shape[:-1]) + (tb.rows,), dtype=out_dtype)
    ws, ws_bytes = _workspace(out, "lrq_mxfp4_gemm_workspace", ctypes.byref(ta), ctypes.byref(tb))
    with _on(a.device):
        call("lrq_mxfp4_gemm", ctypes.byref(ta), ctypes.byref(tb), _p(out), b.rows, f32, _p(ws), ws_bytes,
             _stream(a.device))
    return out


def _workspace(like: torch.Tensor, query: str, *args):
    n = call_raw(query, *args)
    if n < 0:
        check(n, query)
    return (like.new_empty(n // 4, dtype=torch.float32) if n else None), n


def _operand(x: torch.Tensor, cols: int, name: str):
    """x as rows of whole 16-byte pieces (zeros appended where the width is no multiple of 8)."""
    _require_device(x)
    if x.dtype != torch.bfloat16 or x.dim() < 1 or x.shape[-1] != cols:
        raise ValueError(f"{name} must be bf16 [..., {cols}], got {x.dtype} {tuple(x.shape)}")
    if cols == 0:
        return x, x.numel(), 0
    if cols % 8:
        x = torch.nn.functional.pad(x, (0, -cols % 8))
    x2, rows, _, ld = _rows(x, name)
    if ld % 8 or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
        ld = x2.shape[-1]
    return x2, rows, ld


def _product(name: str, x: torch.Tensor, w: MXFP4Tensor, out_dtype, transposed: int) -> torch.Tensor:
    f32 = _out_fp32(out_dtype)
    t = _matrix(w, x.device)
    depth, cols = (w.rows, w.cols) if transposed else (w.cols, w.rows)
    x2, rows, ld = _operand(x, depth, "dy" if transposed else "x")
    out = x.new_empty((x.shape[0], cols) if x.dim() == 2 else x.shape[:-1] + (cols,), dtype=out_dtype)
    if depth == 0:
        return out.zero_()
    ws, ws_bytes = _workspace(out, "lrq_mxfp4_linear_workspace", rows, ctypes.byref(t), transposed)
    with _on(x.device):
        call(name, _p(x2), ld, rows, ctypes.byref(t), _p(out), cols, f32, _p(ws), ws_bytes, _stream(x.device))
    return out


def mxfp4_linear(x: torch.Tensor, w: MXFP4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x @ w^T for bf16 x [..., K] and an MXFP4 weight [N, K]: [..., N], fp32 accumulate."""
    return _product("lrq_mxfp4_linear", x, w, out_dtype, 0)


def mxfp4_linear_backward(dy: torch.Tensor, w: MXFP4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """dy @ w for bf16 dy [..., N] and an MXFP4 weight [N, K]: the gradient of ``mxfp4_linear`` for x."""
    return _product("lrq_mxfp4_linear_t", dy, w, out_dtype, 1)
