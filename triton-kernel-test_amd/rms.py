"""Root-mean-square norm on the HIP kernels, alone or behind a residual add, with an output of the row's type or in 8 bits.

``rms_norm_forward`` / ``add_rms_norm_forward`` / ``rms_norm_backward`` return what they computed; ``autograd.rms_norm``,
``autograd.add_rms_norm`` and ``autograd.rms_norm_linear`` are the same inside autograd.  x is bf16, fp16 or fp32 [..., n]
of any row width and row stride, the weight is of any of the three types; sums and statistics are fp32, each output is
rounded once.  The squares are summed in fp32: rows with elements above 1e19 are out of its range.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import call
from .api import _on, _p, _require_device, _stream
from .fp8 import _empty
from .norm import _dtype, _like, _new, _rows, _weights

__all__ = ["rms_norm_forward", "add_rms_norm_forward", "rms_norm_backward"]


def _forward(x, residual, weight, eps, fp8: bool, add: bool):
    _require_device(x, residual, weight)
    dt = _dtype(x, "x")
    x2, rows, n, ldx = _rows(x, "x")
    device, r2, ldr, w, wdt = x.device, None, 0, None, _lib.LRQ_F32
    if residual is not None:
        _like(residual, x, "residual")
        r2, ldr = _rows(residual, "residual")[::3]
    if weight is not None:
        w, _, wdt = _weights(weight, None, n, device)
    h = _new(x) if add else None
    if fp8:
        y, t = _empty(x, rows, n, x.shape, 1)
        py, pq = None, ctypes.byref(t)
    else:
        y = _new(x)
        py, pq = y.data_ptr(), None
    rstd = x.new_empty(rows if x.dim() == 2 else x.shape[:-1], dtype=torch.float32)  # (an int is 0.8 us less than a shape)
    with _on(device):
        call("lrq_rms_norm_fwd", x2.data_ptr(), ldx, _p(r2), ldr, dt, _p(w), wdt, rows, n, eps, _p(h), n, py, n, pq,
             rstd.data_ptr(), _stream(device))
    return y, h, rstd


def rms_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, fp8: bool = False):
    """(y, rstd) of y = x * rstd * weight over the last axis, rstd = 1 / sqrt(mean(x^2) + eps), fp32 of x's leading
    shape.  ``fp8``: y is an ``FP8Tensor`` (block 1), quantised from its fp32 values."""
    y, _, rstd = _forward(x, None, weight, eps, fp8, False)
    return y, rstd


def add_rms_norm_forward(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                         eps: float = 1e-6, fp8: bool = False):
    """(y, h, rstd): h = residual + x (rounded to x's dtype), y = rms_norm(h), in one pass; ``fp8`` as in
    ``rms_norm_forward``."""
    if residual is None:
        raise ValueError("add_rms_norm_forward needs a residual")
    return _forward(x, residual, weight, eps, fp8, True)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor,
                      dh: Optional[torch.Tensor] = None, weight_grad: bool = True):
    """(dx, dweight) of ``rms_norm_forward`` (h: its x) or ``add_rms_norm_forward`` from dy and dh, the gradient of h from
    its other uses; dx is the gradient for x and for the residual.  dweight is None with ``weight_grad=False`` (a frozen
    weight: its sum is not taken) and fp32 without a weight.  The sum over the rows runs in an order that depends on the shape
    alone."""
    _require_device(dy, dh, h, weight, rstd)
    dt = _dtype(h, "x")
    _like(dy, h, "dy")
    _like(dh, h, "dh")
    if rstd.dtype is not torch.float32 or rstd.shape != h.shape[:-1] or rstd.device != h.device:
        raise ValueError(f"rstd must be fp32 {tuple(h.shape[:-1])} on {h.device}")
    rstd = rstd.contiguous()
    dy2, rows, n, lddy = _rows(dy, "dy")
    h2, _, _, ldh = _rows(h, "x")
    dh2, lddh = (None, 0) if dh is None else _rows(dh, "dh")[::3]
    w, _, wdt = _weights(weight, None, n, h.device)
    dx = _new(h)
    dw = ws = None
    ws_bytes = 0
    if weight_grad:
        ws_bytes = _lib.call_raw("lrq_rms_norm_bwd_workspace", rows, n)
        if ws_bytes < 0:
            _lib.check(ws_bytes, "lrq_rms_norm_bwd_workspace")
        ws = h.new_empty(max(ws_bytes // 4, 1), dtype=torch.float32)
        dw = h.new_empty(n, dtype=torch.float32) if w is None else torch.empty_like(w)
    with _on(h.device):
        call("lrq_rms_norm_bwd", _p(dy2), lddy, _p(dh2), lddh, _p(h2), ldh, dt, _p(w), wdt, _p(rstd), rows, n, _p(dx), n,
             _p(dw), _p(ws), ws_bytes, _stream(h.device))
    return dx, dw
