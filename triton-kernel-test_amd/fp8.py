"""8-bit floating point (OCP e4m3) with one power-of-two scale for a block of 128: quantisation and products.

Activations take a scale for 128 columns of a row (block 1), weights one for 128 x 128 (block 128).  The scales are E8M0
exponents, which the matrix instructions multiply by themselves.  ``fp8_linear`` multiplies activations (quantised on the way,
or an ``FP8Tensor`` such as the norm's) by a weight, ``fp8_linear_backward`` is its gradient for them and
``fp8_weight_gradient`` that for a weight that is trained; ``fp8_gemm`` multiplies two ``FP8Tensor``s.  All accumulate in
fp32, but each eight neighbouring products along the contraction are added in a window: what lies below 2^-13 of the largest
one's power of two is dropped, up to 7 * 2^-13 of that product (normal operands: 1.5e-5 of the output in the mean square).
``autograd.fp8_linear``, ``autograd.rms_norm_linear`` and ``autograd.lora_linear_compressed`` (an ``FP8Tensor`` as its base
weight) call them.
"""

from __future__ import annotations

import ctypes
import math
from typing import Union

import torch

from . import _lib
from ._lib import LrqFp8, call, call_raw, check
from .api import _on, _p, _require_device, _stream
from .norm import _DTYPE, _dtype, _rows

__all__ = ["FP8Tensor", "fp8_from_parts", "fp8_quantize", "fp8_quantize_both", "fp8_dequantize", "fp8_gemm", "fp8_linear",
           "fp8_linear_backward", "fp8_weight_gradient"]

_BYTES = (torch.uint8, torch.float8_e4m3fn, torch.float8_e8m0fnu)


class FP8Tensor:
    """A tensor [..., cols] in e4m3; rows are its leading dimensions flattened.

    ``codes`` uint8 or float8_e4m3fn [rows, >= 128 ceil(cols / 128)], 0 past ``cols``.  ``scales`` uint8 or float8_e8m0fnu:
    one E8M0 exponent for 128 columns of ``block`` (1 or 128) rows, [ceil(rows / block), >= ceil(cols / 128) rounded up to
    4]."""

    # What the library makes lies in one allocation, codes first, whose views are taken when they are asked for: a call on few
    # rows is bound by the host, and an allocation and two views are 3 us of it.
    __slots__ = ("_codes", "_scales", "shape", "block", "_buf")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, block: int = 1):
        self._codes, self._scales, self.shape, self.block, self._buf = codes, scales, tuple(shape), block, None

    def _views(self):
        c, steps, wide = self._buf, _steps(self.shape[-1]), _wide(self.shape[-1])
        rows = math.prod(self.shape[:-1])
        tall = (rows + self.block - 1) // self.block
        self._codes = c.as_strided((rows, 128 * steps), (128 * steps, 1)).view(torch.float8_e4m3fn)
        self._scales = c.as_strided((tall, wide), (wide, 1), c.storage_offset() + rows * 128 * steps)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._views()
        return self._codes

    @codes.setter
    def codes(self, t: torch.Tensor):
        self._scales, self._codes, self._buf = self.scales, t, None

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._views()
        return self._scales

    @scales.setter
    def scales(self, t: torch.Tensor):
        self._codes, self._scales, self._buf = self.codes, t, None

    def __repr__(self) -> str:
        return f"FP8Tensor(shape={self.shape}, block={self.block}, device={self.device})"

    @property
    def rows(self) -> int:
        return math.prod(self.shape[:-1])

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def device(self) -> torch.device:
        return (self._codes if self._buf is None else self._buf).device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def to(self, device) -> "FP8Tensor":
        return FP8Tensor(self.codes.to(device), self.scales.to(device), self.shape, self.block)

    def descriptor(self) -> LrqFp8:
        shape, block, buf = self.shape, self.block, self._buf
        cols = shape[-1] if len(shape) else 0
        if cols <= 0:
            raise ValueError("an FP8 tensor needs rows of at least one element")
        if block != 1 and block != 128:
            raise ValueError(f"a scale is for 1 or 128 rows, got {block}")
        rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
        steps = (cols + 127) // 128
        wide = (steps + 3) // 4 * 4
        if buf is not None:
            p = buf.data_ptr()
            return LrqFp8(p, 128 * steps, p + rows * 128 * steps, wide, rows, cols, block)
        c, s = self._codes, self._scales
        tall = (rows + block - 1) // block
        if not (c.is_cuda and s.is_cuda):
            _require_device(c, s)
        if c.dim() == 2 and s.dim() == 2 and c.dtype in _BYTES and s.dtype in _BYTES and c.device == s.device:
            (cr, cw), (sr, sw), (ldc, c1), (lds, s1) = c.shape, s.shape, c.stride(), s.stride()
            if cr == rows and sr == tall and cw >= 128 * steps and sw >= wide and c1 == 1 and s1 == 1:
                if rows <= 1:  # the stride of a single row means nothing
                    ldc = 128 * steps
                if tall <= 1:
                    lds = wide
                return LrqFp8(c.data_ptr(), ldc, s.data_ptr(), lds, rows, cols, block)
        raise ValueError(f"codes and scales must be bytes [{rows}, >= {128 * steps}] and [{tall}, >= {wide}] with unit inner "
                         f"stride on one device, got {c.dtype} {tuple(c.shape)} on {c.device} and {s.dtype} "
                         f"{tuple(s.shape)} on {s.device}")


def _steps(cols: int) -> int:
    return (cols + 127) // 128


def _wide(cols: int) -> int:
    return (_steps(cols) + 3) // 4 * 4


def _empty(like: torch.Tensor, rows: int, cols: int, shape, block: int) -> tuple[FP8Tensor, LrqFp8]:
    """An FP8 tensor to be written, and its descriptor."""
    steps = (cols + 127) // 128
    wide, codes = (steps + 3) // 4 * 4, rows * 128 * steps
    q = FP8Tensor.__new__(FP8Tensor)
    q._codes = q._scales = None
    q.shape, q.block = tuple(shape), block
    q._buf = buf = like.new_empty(codes + (rows if block == 1 else (rows + 127) // 128) * wide, dtype=torch.uint8)
    p = buf.data_ptr()
    return q, LrqFp8(p, 128 * steps, p + codes, wide, rows, cols, block)


def fp8_from_parts(codes: torch.Tensor, scales: torch.Tensor, block: int = 128) -> FP8Tensor:
    """An ``FP8Tensor`` from a matrix of e4m3 codes [rows, cols] and its scales [ceil(rows / block), ceil(cols / 128)], as a
    checkpoint holds them: E8M0 exponents, or fp32 factors, which must be powers of two from 2^-127 to 2^127.  Copies
    what is not laid out as needed; reads the scales back once if they are fp32."""
    _require_device(codes, scales)
    if codes.dim() != 2 or codes.dtype not in (torch.uint8, torch.float8_e4m3fn) or codes.shape[1] == 0:
        raise ValueError(f"codes must be a matrix of e4m3 bytes, got {codes.dtype} {tuple(codes.shape)}")
    if block != 1 and block != 128:
        raise ValueError(f"a scale is for 1 or 128 rows, got {block}")
    rows, cols = codes.shape
    steps = (cols + 127) // 128
    tall = (rows + block - 1) // block
    if tuple(scales.shape) != (tall, steps) or scales.device != codes.device:
        raise ValueError(f"scales must be [{tall}, {steps}] on {codes.device}, got {tuple(scales.shape)} on {scales.device}")
    if scales.dtype == torch.float32:
        m, e = torch.frexp(scales)  # 2^-127 has no normal fp32, but frexp takes it apart all the same
        if not bool(((m == 0.5) & (e >= -126) & (e <= 128)).all()):
            raise ValueError("fp32 scales must be powers of two from 2^-127 to 2^127: quantise the dequantised weight instead")
        scales = (e + 126).to(torch.uint8)
    elif scales.dtype not in (torch.uint8, torch.float8_e8m0fnu):
        raise ValueError(f"scales must be E8M0 bytes or fp32, got {scales.dtype}")
    c, s = codes.view(torch.uint8), scales.view(torch.uint8)
    if cols % 128 or c.stride(1) != 1 or c.stride(0) % 16 or c.stride(0) < cols or c.data_ptr() % 16:
        c = torch.nn.functional.pad(c, (0, -cols % 128)).clone(memory_format=torch.contiguous_format)
    if steps % 4 or s.stride(1) != 1 or s.stride(0) % 4 or s.stride(0) < steps or s.data_ptr() % 4:
        s = torch.nn.functional.pad(s, (0, -steps % 4)).clone(memory_format=torch.contiguous_format)
    return FP8Tensor(c.view(torch.float8_e4m3fn), s, (rows, cols), block)


def fp8_quantize(x: torch.Tensor, block: int = 1, transpose: bool = False) -> FP8Tensor:
    """x[..., n] (bf16, fp16 or fp32) in e4m3: per block of 128 columns of a row, or with ``block=128`` of 128 rows by 128
    columns, the smallest power of two that the largest magnitude exceeds at most 448 times; elements rounded to the nearest
    code (ties to the even one).  A block with an infinity or a NaN becomes NaN.  ``transpose``: the transpose [n, rows], in
    blocks of 128 of its columns."""
    _require_device(x)
    dt = _dtype(x, "x")
    if block != 1 and block != 128:
        raise ValueError(f"a scale is for 1 or 128 rows, got {block}")
    if transpose and block != 1:
        raise ValueError("the transpose takes blocks of one row")
    x2, rows, n, ldx = _rows(x, "x")
    if transpose:
        if rows == 0:
            raise ValueError("the transpose of no rows has rows of no elements")
        q, t = _empty(x, n, rows, (n, rows), 1)
    else:
        q, t = _empty(x, rows, n, x.shape, block)
    with _on(x.device):
        call("lrq_fp8_quantize", _p(x2), ldx, dt, ctypes.byref(t), int(transpose), _stream(x.device))
    return q


def fp8_quantize_both(x: torch.Tensor) -> tuple[FP8Tensor, FP8Tensor]:
    """(``fp8_quantize(x)``, ``fp8_quantize(x, transpose=True)``) from one read of x: what a product and its weight's gradient
    take."""
    _require_device(x)
    dt = _dtype(x, "x")
    x2, rows, n, ldx = _rows(x, "x")
    if rows == 0:
        raise ValueError("the transpose of no rows has rows of no elements")
    q, t = _empty(x, rows, n, x.shape, 1)
    qt, tt = _empty(x, n, rows, (n, rows), 1)
    with _on(x.device):
        call("lrq_fp8_quantize_both", x2.data_ptr(), ldx, dt, ctypes.byref(t), ctypes.byref(tt), _stream(x.device))
    return q, qt


def fp8_dequantize(q: FP8Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of q, rounded to dtype (exact in fp32, and in bf16 but for its subnormal numbers)."""
    t = q.descriptor()
    out = (q._codes if q._buf is None else q._buf).new_empty(q.shape, dtype=dtype)
    with _on(q.device):
        call("lrq_fp8_dequantize", ctypes.byref(t), _p(out), q.cols, _dtype(out, "the output"), _stream(q.device))
    return out


def _out_dtype(dtype: torch.dtype) -> int:
    d = _DTYPE.get(dtype)
    if d is None:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {dtype}")
    return d


def _out(x: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """x's leading shape and cols, to be written (sizes one by one: 0.5 us less than a tuple of them)."""
    return x.new_empty(rows, cols, dtype=dtype) if x.dim() == 2 else x.new_empty(x.shape[:-1] + (cols,), dtype=dtype)


def _matrix(w: FP8Tensor, device: torch.device) -> LrqFp8:
    if not isinstance(w, FP8Tensor) or len(w.shape) != 2:
        raise ValueError("the weight must be an FP8Tensor of two dimensions")
    if w.device != device:
        raise ValueError(f"the weight is on {w.device}, the operand on {device}")
    return w.descriptor()


def _product(name: str, a: FP8Tensor, tb: LrqFp8, cols: int, out_dtype, nn: int) -> torch.Tensor:
    dt = _out_dtype(out_dtype)
    ta = a.descriptor()
    rows, any_ = ta.rows, a._codes if a._buf is None else a._buf
    if len(a.shape) == 2:
        out = any_.new_empty(rows, cols, dtype=out_dtype)
    else:
        out = any_.new_empty(a.shape[:-1] + (cols,), dtype=out_dtype)
    device, pa, pb, ws, n = out.device, ctypes.byref(ta), ctypes.byref(tb), None, 0
    if nn or rows > 16:  # (fewer rows split nothing over workgroups)
        n = call_raw("lrq_fp8_gemm_workspace", pa, pb, nn)
        if n < 0:
            check(n, "lrq_fp8_gemm_workspace")
        ws = out.new_empty(n // 4, dtype=torch.float32) if n else None
    with _on(device):
        call(name, pa, pb, out.data_ptr(), cols, dt, _p(ws), n, _stream(device))
    return out


def _quantize_product(x: torch.Tensor, name: str, tb: LrqFp8, cols: int, out_dtype, nn: int) -> torch.Tensor:
    """x quantised and multiplied in one call: of 37 rows 14.3 us of the host, in two 18.6."""
    dt, odt = _dtype(x, name), _out_dtype(out_dtype)
    x2, rows, _, ldx = _rows(x, name)
    pb = ctypes.byref(tb)
    n = call_raw("lrq_fp8_quantize_gemm_workspace", rows, pb, nn)
    if n < 0:
        check(n, "lrq_fp8_quantize_gemm_workspace")
    out = _out(x, rows, cols, out_dtype)
    ws = x.new_empty(n, dtype=torch.uint8)
    with _on(x.device):
        call("lrq_fp8_quantize_gemm", x2.data_ptr(), ldx, dt, rows, pb, nn, out.data_ptr(), cols, odt, ws.data_ptr(), n,
             _stream(x.device))
    return out


def fp8_gemm(a: FP8Tensor, b: FP8Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a @ b^T for a [..., K] and b [N, K], both e4m3 of any block: [..., N], fp32 accumulate."""
    tb = _matrix(b, a.device)
    if a.cols != b.cols:
        raise ValueError(f"operands have {a.cols} and {b.cols} columns")
    return _product("lrq_fp8_gemm", a, tb, b.rows, out_dtype, 0)


def fp8_linear(x: Union[torch.Tensor, FP8Tensor], w: FP8Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x @ w^T for an e4m3 weight [N, K] and x [..., K], an ``FP8Tensor`` or bf16, fp16 or fp32 that is quantised (block 1) on
    the way: [..., N], fp32 accumulate."""
    if isinstance(x, FP8Tensor):
        return fp8_gemm(x, w, out_dtype)
    t = _matrix(w, x.device)
    _require_device(x)
    dt, k = _dtype(x, "x"), t.cols
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {tuple(x.shape)}")
    if dt == _lib.LRQ_F32 or k % 8 or x.numel() > _lib.LRQ_FP8_LINEAR_ROWS * k:
        return _quantize_product(x, "x", t, t.rows, out_dtype, 0)
    odt = _out_dtype(out_dtype)
    x2, rows, _, ldx = _rows(x, "x")
    out = _out(x, rows, t.rows, out_dtype)
    with _on(x.device):
        call("lrq_fp8_linear", _p(x2), ldx, dt, rows, ctypes.byref(t), _p(out), t.rows, odt, _stream(x.device))
    return out


def fp8_linear_backward(dy: Union[torch.Tensor, FP8Tensor], w: FP8Tensor,
                        out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """dy @ w for an e4m3 weight [N, K] of block 128 and dy [..., N] (quantised on the way, block 1, if it is not an
    ``FP8Tensor``): the gradient of ``fp8_linear`` for x."""
    t = _matrix(w, dy.device)
    if t.block != 128:
        raise ValueError("the gradient needs a weight with a scale for 128 rows")
    if len(dy.shape) < 1 or dy.shape[-1] != t.rows:
        raise ValueError(f"dy must be [..., {t.rows}], got {tuple(dy.shape)}")
    if t.rows == 0:
        _require_device(dy)
        _out_dtype(out_dtype)
        return dy.new_zeros(dy.shape[:-1] + (t.cols,), dtype=out_dtype)
    if isinstance(dy, FP8Tensor):
        return _product("lrq_fp8_gemm_nn", dy, t, t.cols, out_dtype, 1)
    _require_device(dy)
    return _quantize_product(dy, "dy", t, t.cols, out_dtype, 1)


def fp8_weight_gradient(dy: torch.Tensor, x: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """dy^T @ x for dy [..., N] and x [..., K], both quantised along their rows (blocks of 128 tokens): [N, K], the gradient
    of ``fp8_linear`` for a weight that is trained."""
    _require_device(dy, x)
    if dy.dim() < 1 or x.dim() < 1 or dy.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"dy and x must have the same leading dimensions, got {tuple(dy.shape)} and {tuple(x.shape)}")
    if dy.device != x.device:
        raise ValueError(f"dy is on {dy.device}, x on {x.device}")
    _out_dtype(out_dtype)
    if x.numel() == 0 or dy.numel() == 0:  # no tokens
        return x.new_zeros((dy.shape[-1], x.shape[-1]), dtype=out_dtype)
    return fp8_gemm(fp8_quantize(dy, transpose=True), fp8_quantize(x, transpose=True), out_dtype)
