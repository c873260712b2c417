"""Layer norm and dropout on the HIP kernels: the operators in front of a compressed layer (the
reference has none; its profiles run a LoRA layer alone).

``layer_norm_forward`` / ``layer_norm_backward`` and the fused ``dropout_add_layer_norm_forward`` /
``_backward`` return what they computed; ``autograd.layer_norm``, ``autograd.dropout`` and
``autograd.dropout_add_layer_norm`` are the same inside autograd.  x is bf16, fp16 or fp32 [..., n] of any row
width and row stride, weights are of any of the three types; sums and statistics are fp32, each output
is rounded once.

Dropout's mask is a function of (seed, offset, row, column) and is never stored: ``dropout`` of the
gradient with the same seed is the backward pass.  ``seed`` is an int, a pair (seed, offset), or an int64
device tensor of those two words, alone or with a further offset as (tensor, offset): such a tensor
is read when the kernel runs, so a captured graph draws a new mask in each replay if its second word is
advanced in between (give each dropout of the graph an offset of its own).  With p = 0 it may be None.  An element
takes 16 random bits: p is rounded to a multiple of 1 / 65536 (at least one for p > 0, at most 65535 for p < 1).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import LrqDropout, call
from .api import _on, _p, _require_device, _rows_view, _stream

__all__ = ["layer_norm_forward", "layer_norm_backward", "dropout", "dropout_add_layer_norm_forward",
           "dropout_add_layer_norm_backward"]

_DTYPE = {torch.bfloat16: _lib.LRQ_BF16, torch.float16: _lib.LRQ_F16, torch.float32: _lib.LRQ_F32}


def _dtype(t: torch.Tensor, name: str) -> int:
    d = _DTYPE.get(t.dtype)
    if d is None:
        raise ValueError(f"{name} must be bf16, fp16 or fp32, got {t.dtype}")
    return d


# Small batches are bound by the host (a call of a few rows: 10 us for 3 us of kernel), so the usual case, contiguous
# operands, takes as few torch calls as it can: no views, empty_like and new_empty for the outputs (half of empty's time).
def _rows(x: torch.Tensor, name: str) -> tuple[torch.Tensor, int, int, int]:
    """x as rows: (a tensor to take the pointer of, rows, row width, row stride); rows do not overlap (an expanded
    gradient is copied)."""
    n = x.shape[-1] if x.dim() else 0
    if n == 0:
        raise ValueError(f"{name} must have rows of at least one element")
    if x.is_contiguous():
        return x, x.numel() // n, n, n
    x2, rows, n, ld = _rows_view(x)
    if ld < n:
        if rows > 1:
            x2 = x2.contiguous()
        ld = n
    return x2, rows, n, ld


def _like(t: Optional[torch.Tensor], x: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    if t is not None and (t.shape != x.shape or t.dtype is not x.dtype or t.device != x.device):
        raise ValueError(f"{name} must be {x.dtype} {tuple(x.shape)} on {x.device}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t


def _new(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _weights(weight, bias, n: int, device: torch.device):
    """(weight, bias, their dtype) ready for the kernels."""
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.dim() != 1 or t.shape[0] != n or t.device != device):
            raise ValueError(f"{name} must be [{n}] on {device}, got {tuple(t.shape)} on {t.device}")
    if weight is None:
        if bias is None:
            return None, None, _lib.LRQ_F32
        return None, bias.contiguous(), _dtype(bias, "bias")
    if bias is not None:
        if bias.dtype is not weight.dtype:
            raise ValueError("weight and bias must have one dtype")
        bias = bias.contiguous()
    return weight.contiguous(), bias, _dtype(weight, "weight")


def _statistics(mean: torch.Tensor, rstd: torch.Tensor, x: torch.Tensor):
    lead, device = x.shape[:-1], x.device
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype is not torch.float32 or t.shape != lead or t.device != device:
            raise ValueError(f"{name} must be fp32 {tuple(lead)} on {device}")
    return mean.contiguous(), rstd.contiguous()


def _keep(p: float) -> int:
    p = float(p)
    if not 0.0 <= p <= 1.0:  # (also refuses NaN)
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    drop = round(65536 * p)
    if 0.0 < p < 1.0:
        drop = min(max(drop, 1), 65535)
    return 65536 - drop


def _drop(p: float, seed, device: torch.device) -> tuple[LrqDropout, Optional[torch.Tensor]]:
    """The descriptor and the state tensor it points to (kept by the caller until the launch)."""
    keep = _keep(p)
    state, offset = None, 0
    if isinstance(seed, (tuple, list)):
        if len(seed) != 2:
            raise ValueError("seed must be an int, a tensor, or a pair with an offset")
        seed, offset = seed
    if isinstance(seed, torch.Tensor):
        state, seed = seed, 0
        if state.dtype != torch.int64 or state.numel() != 2 or state.device != device or not state.is_contiguous():
            raise ValueError(f"a seed tensor must be two contiguous int64 words on {device}")
    if seed is None and keep == 65536:  # nothing is drawn
        seed = 0
    if isinstance(seed, bool) or not isinstance(seed, int) or isinstance(offset, bool) or not isinstance(offset, int):
        raise ValueError("seed and offset must be ints")
    m = (1 << 64) - 1
    return LrqDropout(keep, seed & m, offset & m, None if state is None else state.data_ptr()), state


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd) of y = (x - mean) * rstd * weight + bias over the last axis; mean and rstd are fp32
    of x's leading shape."""
    _require_device(x, weight, bias)
    dt = _dtype(x, "x")
    x2, rows, n, ldx = _rows(x, "x")
    w, b, wdt = _weights(weight, bias, n, x.device)
    y = _new(x)
    mean = x.new_empty((rows,) if x.dim() == 2 else x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    with _on(x.device):
        call("lrq_layer_norm_fwd", None, _p(x2), ldx, None, 0, dt, _p(w), _p(b), wdt, rows, n, eps, None, 0, _p(y), n,
             _p(mean), _p(rstd), _stream(x.device))
    return y, mean, rstd


def _backward(drop, dy, dh, h, weight, mean, rstd, weight_grad: bool, fused: bool, want_dx: bool):
    dt = _dtype(h, "x")
    _like(dy, h, "dy")
    _like(dh, h, "dh")
    mean, rstd = _statistics(mean, rstd, h)
    dy2, rows, n, lddy = _rows(dy, "dy")
    w, _, wdt = _weights(weight, None, n, h.device)
    h2, _, _, ldh = _rows(h, "x")
    dh2, lddh = (None, 0) if dh is None else _rows(dh, "dh")[::3]
    dx = _new(h) if want_dx else None
    dres = _new(h) if fused else None
    dw = db = ws = None
    ws_bytes = 0
    if weight_grad:
        ws_bytes = _lib.call_raw("lrq_layer_norm_bwd_workspace", rows, n)
        if ws_bytes < 0:
            _lib.check(ws_bytes, "lrq_layer_norm_bwd_workspace")
        ws = h.new_empty(max(ws_bytes // 4, 1), dtype=torch.float32)
        dw = h.new_empty(n, dtype=torch.float32) if w is None else torch.empty_like(w)
        db = torch.empty_like(dw)
    with _on(h.device):
        call("lrq_layer_norm_bwd", drop, _p(dy2), lddy, _p(dh2), lddh, _p(h2), ldh, dt, _p(w), wdt, _p(mean), _p(rstd),
             rows, n, _p(dx), n, _p(dres), n, _p(dw), _p(db), _p(ws), ws_bytes, _stream(h.device))
    return dx, dres, dw, db


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, weight_grad: bool = True):
    """(dx, dweight, dbias) of ``layer_norm_forward``; the last two are None with ``weight_grad=False``
    (frozen weights: their sums are not taken).  Without a weight they are fp32.  The sums over the rows run in an order that
    depends on the shape alone."""
    _require_device(dy, x, weight, mean, rstd)
    dx, _, dw, db = _backward(None, dy, None, x, weight, mean, rstd, weight_grad, False, True)
    return dx, dw, db


def dropout(x: torch.Tensor, p: float, seed, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + (kept ? x / (1 - p) : 0), rounded once; ``dropout(dy, p, seed)`` is its gradient for x."""
    _require_device(x, residual)
    dt = _dtype(x, "x")
    _like(residual, x, "residual")
    drop, _state = _drop(p, seed, x.device)
    out = _new(x)
    if x.numel() == 0:
        return out
    x2, rows, n, ldx = _rows(x.reshape(1) if x.dim() == 0 else x, "x")
    r2, ldr = (None, 0)
    if residual is not None:
        r2, ldr = _rows(residual.reshape(1) if x.dim() == 0 else residual, "residual")[::3]
    with _on(x.device):
        call("lrq_dropout_add", ctypes.byref(drop), _p(x2), ldx, _p(r2), ldr, dt, rows, n, _p(out), n, _stream(x.device))
    return out


def dropout_add_layer_norm_forward(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor],
                                   bias: Optional[torch.Tensor], p: float, seed, eps: float = 1e-5):
    """(y, h, mean, rstd): h = residual + dropout(x) (rounded to x's dtype), y = layer_norm(h), in one pass."""
    _require_device(x, residual, weight, bias)
    dt = _dtype(x, "x")
    _like(residual, x, "residual")
    x2, rows, n, ldx = _rows(x, "x")
    r2, ldr = (None, 0) if residual is None else _rows(residual, "residual")[::3]
    w, b, wdt = _weights(weight, bias, n, x.device)
    drop, _state = _drop(p, seed, x.device)
    y = _new(x)
    h = _new(x)
    mean = x.new_empty((rows,) if x.dim() == 2 else x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    with _on(x.device):
        call("lrq_layer_norm_fwd", ctypes.byref(drop), _p(x2), ldx, _p(r2), ldr, dt, _p(w), _p(b), wdt, rows, n, eps, _p(h),
             n, _p(y), n, _p(mean), _p(rstd), _stream(x.device))
    return y, h, mean, rstd


def dropout_add_layer_norm_backward(dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor,
                                    weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, p: float, seed,
                                    weight_grad: bool = True):
    """(dx, dresidual, dweight, dbias) of ``dropout_add_layer_norm_forward`` from dy and dh (the gradient of h
    from its other uses, or None).  With p = 0 dx and dresidual are one tensor."""
    _require_device(dy, dh, h, weight, mean, rstd)
    drop, _state = _drop(p, seed, h.device)
    some = drop.keep < 65536
    dx, dres, dw, db = _backward(ctypes.byref(drop), dy, dh, h, weight, mean, rstd, weight_grad, True, some)
    return (dx if some else dres), dres, dw, db
