"""Compress-on-save: the compressed format inside autograd.

The reference's system profiles run the path between a LoRA layer's forward and its
gradient: ``compute_lora`` (low_rank_system_profile_forward.py:8-12) produces y, the
activation x is compressed (``:50``), and before ``compute_lora_gradient`` (``:14-18``) it is
decompressed again (low_rank_system_profile_backward.py:55-61).  This module makes that
round trip part of autograd:

* ``compute_lora`` / ``compute_lora_gradient`` keep the reference's formulas (the weight is a
  dense [out, in] tensor here; the reference passes a Linear module to the forward).
* ``LoRALinearCompressed`` is an autograd Function whose forward is ``compute_lora`` and which
  saves x in the compressed format; its backward returns dx, dA and dB of
  ``compute_lora_gradient`` (W is frozen, as in the reference's LoRA setting).  With
  ``fused=True`` (the default) x is never decoded: dA = x^T (dy B^T) and x A come from the codes,
  in one pass for both (``lora_grads``: int4 / g64 / rank 16, LoRA rank 16) or from the
  transposed dequant-GEMM and the dequant-GEMM (LoRA rank 16 or 32, plain format); otherwise,
  or for other shapes, x is decoded and the formulas run on it.
* ``compressed_saved_tensors`` is a ``torch.autograd.graph.saved_tensors_hooks`` context that
  stores every saved bf16 activation with a suitable last dimension in the compressed format
  and decodes it when backward asks for it, for any model.
* ``layer_norm``, ``dropout``, ``dropout_add_layer_norm`` and ``mxfp4_linear`` are the operators of
  ``norm.py`` and ``mxfp4.py`` with their gradients, ``rms_norm``, ``add_rms_norm``, ``fp8_linear`` and
  ``rms_norm_linear`` those of ``rms.py`` and ``fp8.py``; ``lora_linear_compressed`` takes an MXFP4 or
  8-bit base weight and LoRA dropout.
* ``fit_basis`` builds the rank-r basis V from a sample of activation rows (top right singular
  vectors), the counterpart of the reference's low-rank factors of x.

The compression is lossy: gradients are those of the decoded activations.
"""

from __future__ import annotations

from typing import Callable, Optional

import torch
from torch.autograd.function import once_differentiable

from . import fp8 as _f8
from . import mxfp4 as _mx
from . import norm as _norm
from . import rms as _rms
from .api import CompressedActivation, LowRankBasis, decode, encode, lora_grads

__all__ = ["compute_lora", "compute_lora_gradient", "LoRALinearCompressed", "lora_linear_compressed",
           "compressed_saved_tensors", "fit_basis", "layer_norm", "dropout", "dropout_add_layer_norm", "mxfp4_linear",
           "rms_norm", "add_rms_norm", "fp8_linear", "rms_norm_linear"]


def compute_lora(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """y = x W^T + (x A) B (low_rank_system_profile_forward.py:8-12; W [out, in]).  Leading
    dimensions are folded into the rows, so every product is a plain 2-D GEMM."""
    x2 = _flat(x)
    y = x2 @ w.mT + (x2 @ a) @ b
    return y.reshape(x.shape[:-1] + (w.shape[0],))


def compute_lora_gradient(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, a: torch.Tensor,
                          b: torch.Tensor):
    """(dx, dA, dB) of ``compute_lora`` (low_rank_system_profile_forward.py:14-18, with the
    weight in [out, in] layout: the reference's ``w.mT`` is W^T's transpose there)."""
    dx = dy @ (w + b.mT @ a.mT)
    da = x.mT @ (dy @ b.mT)
    db = (x @ a).mT @ dy
    return dx, da, db


def _flat(t: torch.Tensor) -> torch.Tensor:
    return t.reshape(-1, t.shape[-1])


class LoRALinearCompressed(torch.autograd.Function):
    """y = compute_lora(x, W, A, B); x is saved compressed (bits, group, optional basis).

    Gradients: dx, dA, dB of compute_lora_gradient on the decoded x; W gets none.  ``fused``
    reads the codes directly for dA and x A (no decoded x), see the module docstring.  W may be an
    ``MXFP4Tensor`` or ``FP8Tensor`` [out, in].  With ``dropout_p`` the LoRA branch reads dropout(x):
    y = x W^T + (dropout(x) A) B, its mask drawn again from ``seed`` in the backward pass, where x is decoded for it."""

    @staticmethod
    def forward(ctx, x, w, a, b, basis: Optional[LowRankBasis], bits: int, group: int, fused: bool = True,
                dropout_p: float = 0.0, seed=None):
        ctx.p, ctx.seed, state = _seeded(dropout_p, seed)
        mx = isinstance(w, (_mx.MXFP4Tensor, _f8.FP8Tensor))
        if ctx.p == 0.0 and not mx:
            y = compute_lora(x, w, a, b)
        else:
            x2 = _flat(x)
            xd = _norm.dropout(x2, ctx.p, seed) if ctx.p > 0.0 else x2
            # the base product in x's type before the branch is added, as compute_lora has it: in fp32 it would be
            # written and read again at twice the bytes
            base = _product(x2, w) if mx else x2 @ w.mT
            y = torch.addmm(base, xd @ a, b).reshape(x.shape[:-1] + (w.shape[0],))
        ctx.c = encode(x.detach(), basis, bits=bits, group_size=group)
        ctx.fused = fused
        ctx.mx, weight = _weight(w) if mx else (None, (w,))
        ctx.save_for_backward(a, b, state, *weight)
        return y

    @staticmethod
    def backward(ctx, dy):
        a, b, state, *weight = ctx.saved_tensors
        w = weight[0] if ctx.mx is None else _saved_weight(ctx.mx, *weight)
        c, ctx.c = ctx.c, None
        dy2 = _flat(dy)
        codes = ctx.fused and ctx.p == 0.0 and _codes_gemm_ok(c, a, dy2)
        if ctx.p == 0.0 and ctx.mx is None:
            if codes:
                dx = dy2 @ (w + b.mT @ a.mT)
                g = dy2 @ b.mT
            else:
                dx, da, db = compute_lora_gradient(dy2, _flat(decode(c)), w, a, b)
        else:
            g = dy2 @ b.mT
            dx = _product_backward(dy2, w) if ctx.mx is not None else dy2 @ w
            if ctx.p > 0.0:
                # (dy W and g A^T rounded to dy's type ahead of their sum, which takes them from memory)
                dx = _norm.dropout(g @ a.mT, ctx.p, _with_state(ctx.seed, state), residual=dx)
            else:
                dx = torch.addmm(dx, g, a.mT)
            if not codes:
                xh = _flat(decode(c))
                if ctx.p > 0.0:
                    xh = _norm.dropout(xh, ctx.p, _with_state(ctx.seed, state))
                da, db = xh.mT @ g, (xh @ a).mT @ dy2
        if codes:
            # x A and x^T (dy B^T) from one pass over the codes where the format allows it
            xa, da = lora_grads(c, a, g, xa_dtype=a.dtype, da_dtype=torch.float32)
            da = da.to(a.dtype)
            db = xa.mT @ dy2  # (x A)^T dy
        dx = dx.reshape(dy.shape[:-1] + (a.shape[0],))
        return dx, None, da, db, None, None, None, None, None, None


def _codes_gemm_ok(c: CompressedActivation, a: torch.Tensor, dy2: torch.Tensor) -> bool:
    """The dequant-GEMMs serve LoRA rank 16 / 32 on the plain (unrotated, no outlier
    channels) format with bf16 operands."""
    return (a.shape[1] in (16, 32) and not c.hadamard and c.idx is None and a.dtype == torch.bfloat16
            and dy2.dtype == torch.bfloat16)


def lora_linear_compressed(x, w, a, b, basis: Optional[LowRankBasis] = None, bits: int = 4, group: int = 64,
                           fused: bool = True, dropout_p: float = 0.0, seed=None):
    """The LoRA layer that saves x compressed (``LoRALinearCompressed``).  w: dense [out, in], an
    ``MXFP4Tensor`` or an ``FP8Tensor`` of block 128; ``dropout_p`` > 0 needs a ``seed`` (``norm.dropout``'s), a new one for
    every step and layer."""
    _frozen(w)
    return LoRALinearCompressed.apply(x, w, a, b, basis, bits, group, fused, dropout_p, seed)


def _seeded(p: float, seed):
    """(p, seed without its tensor, the tensor or None): a seed tensor is saved for the backward pass, which then
    refuses one that was changed in between (it would draw another mask)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if p > 0.0 and seed is None:
        raise ValueError("dropout needs a seed")
    if isinstance(seed, torch.Tensor):
        return p, (None, 0), seed
    if isinstance(seed, (tuple, list)) and len(seed) == 2 and isinstance(seed[0], torch.Tensor):
        return p, (None, seed[1]), seed[0]
    return p, seed, None


def _with_state(seed, state):
    return seed if state is None else (state, seed[1])


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm.layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx, dw, db = _norm.layer_norm_backward(dy, x, weight, mean, rstd, weight_grad=need_w or need_b)
        return dx, dw if need_w else None, db.to(ctx.bias_dtype) if need_b else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis (``norm.layer_norm_forward``) with gradients for x, weight and bias; the sums of
    the weights' gradients are skipped where neither needs one."""
    return _LayerNorm.apply(x, weight, bias, eps)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed):
        ctx.p, ctx.seed, state = _seeded(p, seed)
        ctx.save_for_backward(state)
        return _norm.dropout(x, p, seed, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        state, = ctx.saved_tensors
        dx = _norm.dropout(dy, ctx.p, _with_state(ctx.seed, state)) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout(x: torch.Tensor, p: float, seed, residual: Optional[torch.Tensor] = None,
            training: bool = True) -> torch.Tensor:
    """residual + dropout(x) (``norm.dropout``); the mask is drawn again for the gradient, not stored.  With
    ``training=False`` x itself (plus the residual)."""
    if not training:
        return x if residual is None else x + residual
    return _Dropout.apply(x, residual, p, seed)


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, p, seed, eps):
        ctx.p, ctx.seed, state = _seeded(p, seed)
        y, h, mean, rstd = _norm.dropout_add_layer_norm_forward(x, residual, weight, bias, p, seed, eps)
        ctx.save_for_backward(h, weight, mean, rstd, state)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, weight, mean, rstd, state = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 7
        dy = torch.zeros_like(h) if dy is None else dy
        seed = _with_state(ctx.seed, state)
        _, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        dx, dres, dw, db = _norm.dropout_add_layer_norm_backward(dy, dh, h, weight, mean, rstd, ctx.p, seed,
                                                                 weight_grad=need_w or need_b)
        return (dx, dres if need_r else None, dw if need_w else None, db.to(ctx.bias_dtype) if need_b else None, None,
                None, None)


def dropout_add_layer_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed, eps: float = 1e-5):
    """(y, h) of h = residual + dropout(x), y = layer_norm(h), in one kernel each way; h is the residual stream that
    the next block adds to."""
    return _DropoutAddLayerNorm.apply(x, residual, weight, bias, p, seed, eps)


def _frozen(w):
    """A weight whose backward pass would be refused is refused before the forward one."""
    if isinstance(w, _f8.FP8Tensor) and (len(w.shape) != 2 or w.block != 128):
        raise ValueError(f"the gradient needs a weight with a scale for 128 x 128 of a matrix's elements, got {w}")


def _weight(w):
    """(what the context keeps of an MXFP4 or 8-bit w, the tensors to save): the backward pass refuses a weight changed in
    between.  Tensors made in inference mode carry no version and cannot be saved; such a weight is kept as it is."""
    if w.codes.is_inference() or w.scales.is_inference():
        return w, (None, None)
    return (w.shape, getattr(w, "block", None)), (w.codes, w.scales)


def _saved_weight(kept, codes, scales):
    if codes is None:
        return kept
    shape, block = kept
    return _mx.MXFP4Tensor(codes, scales, shape) if block is None else _f8.FP8Tensor(codes, scales, shape, block)


def _product(x, w):
    return _mx.mxfp4_linear(x, w) if isinstance(w, _mx.MXFP4Tensor) else _f8.fp8_linear(x, w, x.dtype)


def _product_backward(dy, w):
    return (_mx.mxfp4_linear_backward(dy, w) if isinstance(w, _mx.MXFP4Tensor)
            else _f8.fp8_linear_backward(dy, w, dy.dtype))


class _MXFP4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, out_dtype):
        ctx.w, weight = _weight(w)
        ctx.save_for_backward(*weight)
        return _mx.mxfp4_linear(x, w, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        # the product's rows are bf16, a matrix instruction's operand beside the widened weight; dx, of x's type, is bf16 too
        return _mx.mxfp4_linear_backward(dy.to(torch.bfloat16), _saved_weight(ctx.w, *ctx.saved_tensors)), None, None


def mxfp4_linear(x: torch.Tensor, w: "_mx.MXFP4Tensor", out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x w^T for a frozen MXFP4 weight (``mxfp4.mxfp4_linear``), with the gradient for x (taken from dy in bf16)."""
    return _MXFP4Linear.apply(x, w, out_dtype)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        y, rstd = _rms.rms_norm_forward(x, weight, eps)
        ctx.save_for_backward(x, weight, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, rstd = ctx.saved_tensors
        dx, dw = _rms.rms_norm_backward(dy, x, weight, rstd, weight_grad=ctx.needs_input_grad[1])
        return dx, dw, None


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Root-mean-square norm over the last axis (``rms.rms_norm_forward``) with gradients for x and weight; the sum of
    the weight's gradient is skipped where it needs none."""
    return _RmsNorm.apply(x, weight, eps)


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _rms.add_rms_norm_forward(x, residual, weight, eps)
        ctx.save_for_backward(h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:  # the norm's output went unused
            return dh, dh, None, None
        dx, dw = _rms.rms_norm_backward(dy, h, weight, rstd, dh, weight_grad=ctx.needs_input_grad[2])
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """(y, h) of h = residual + x, y = rms_norm(h), in one kernel each way; h is the residual stream that the next block
    adds to."""
    return _AddRmsNorm.apply(x, residual, weight, eps)


class _FP8Linear(torch.autograd.Function):
    """A frozen 8-bit weight."""

    @staticmethod
    def forward(ctx, x, w, out_dtype):
        ctx.w, weight = _weight(w)
        ctx.save_for_backward(*weight)
        ctx.dtype = x.dtype
        return _f8.fp8_linear(x, w, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _f8.fp8_linear_backward(dy, _saved_weight(ctx.w, *ctx.saved_tensors), ctx.dtype), None, None


class _FP8LinearTrained(torch.autograd.Function):
    """A dense weight, quantised here; x is kept for the weight's gradient in 8 bits, as that product reads it."""

    @staticmethod
    def forward(ctx, x, w, out_dtype):
        q = _f8.fp8_quantize(w, 128)
        ctx.shape, ctx.dtype, ctx.w_dtype = q.shape, x.dtype, w.dtype
        ctx.tokens = x.numel() // x.shape[-1] if x.shape[-1] else 0
        xq, xt = _f8.fp8_quantize_both(x) if ctx.needs_input_grad[1] and ctx.tokens else (x, None)
        ctx.save_for_backward(*((q.codes, q.scales) if ctx.needs_input_grad[0] else (None, None)),
                              *((xt.codes, xt.scales) if xt is not None else (None, None)))
        return _f8.fp8_linear(xq, q, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales, xc, xs = ctx.saved_tensors
        dx = dw = dyt = None
        if ctx.needs_input_grad[1] and ctx.tokens and dy.numel():
            dy, dyt = _f8.fp8_quantize_both(dy) if ctx.needs_input_grad[0] else (dy, _f8.fp8_quantize(dy, transpose=True))
        if ctx.needs_input_grad[0]:
            dx = _f8.fp8_linear_backward(dy, _f8.FP8Tensor(codes, scales, ctx.shape, 128), ctx.dtype)
        if ctx.needs_input_grad[1]:
            if dyt is not None:
                dw = _f8.fp8_gemm(dyt, _f8.FP8Tensor(xc, xs, (ctx.shape[1], ctx.tokens), 1), ctx.w_dtype)
            else:
                dw = torch.zeros(ctx.shape, dtype=ctx.w_dtype, device=dy.device)
        return dx, dw, None


def fp8_linear(x: torch.Tensor, w, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x w^T in 8 bits (``fp8.fp8_linear``), of x's type unless ``out_dtype`` says otherwise.  w: an ``FP8Tensor`` of block
    128 (frozen: a gradient for x alone) or a dense [out, in] weight, which is quantised in each call and gets its
    gradient; all products of the backward pass are in 8 bits too."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor of at least one dimension")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if isinstance(w, _f8.FP8Tensor):
        _frozen(w)
        return _FP8Linear.apply(x, w, out_dtype)
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise ValueError("the weight must be an FP8Tensor or a dense matrix")
    if not torch.is_grad_enabled():  # (a parameter asks for its gradient all the same, for which x is quantised along the tokens)
        return _f8.fp8_linear(x, _f8.fp8_quantize(w, 128), out_dtype)
    return _FP8LinearTrained.apply(x, w, out_dtype)


class _RmsNormLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, norm_weight, eps, weights):
        if residual is None:
            q, rstd = _rms.rms_norm_forward(x, norm_weight, eps, fp8=True)
            h = x
        else:
            q, h, rstd = _rms.add_rms_norm_forward(x, residual, norm_weight, eps, fp8=True)
        kept = [_weight(w) for w in weights]
        ctx.w = [k for k, _ in kept]
        ctx.save_for_backward(h, norm_weight, rstd, *(t for _, ts in kept for t in ts))
        ctx.add = residual is not None
        ctx.set_materialize_grads(False)
        y = tuple(_f8.fp8_linear(q, w, x.dtype) for w in weights)
        return y + (h,) if ctx.add else y

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        h, norm_weight, rstd, *saved = ctx.saved_tensors
        dh = grads[len(ctx.w)] if ctx.add else None
        some = [(g, _saved_weight(k, *saved[2 * i:2 * i + 2])) for i, (g, k) in enumerate(zip(grads, ctx.w)) if g is not None]
        if not some:
            return dh, dh if ctx.add else None, None, None, None
        # several products' gradients are added in fp32 and rounded once, as a single one is
        parts = [_f8.fp8_linear_backward(g, w, h.dtype if len(some) == 1 else torch.float32) for g, w in some]
        dn = parts[0]
        for p in parts[1:]:
            dn = dn.add_(p)
        dx, dw = _rms.rms_norm_backward(dn.to(h.dtype), h, norm_weight, rstd, dh, weight_grad=ctx.needs_input_grad[2])
        return dx, dx if ctx.add and ctx.needs_input_grad[1] else None, dw, None, None


def rms_norm_linear(x: torch.Tensor, norm_weight: Optional[torch.Tensor], weights, residual: Optional[torch.Tensor] = None,
                    eps: float = 1e-6):
    """The pre-norm of a layer and the products behind it: n = rms_norm(residual + x), quantised as it leaves the norm,
    times the frozen 8-bit weight(s).  ``weights``: an ``FP8Tensor`` of block 128, or several that share n (query, key and
    value).  Returns a y for each weight (one y for a single FP8Tensor), and with a residual also h = residual + x, last.
    Gradients go to x, the residual and the norm's weight; n itself is not kept."""
    single = isinstance(weights, _f8.FP8Tensor)
    ws = (weights,) if single else tuple(weights)
    if not ws or not all(isinstance(w, _f8.FP8Tensor) for w in ws):
        raise ValueError("weights must be FP8Tensors")
    for w in ws:
        _frozen(w)
    out = _RmsNormLinear.apply(x, residual, norm_weight, eps, ws)
    return out[0] if single and residual is None else out


class compressed_saved_tensors(torch.autograd.graph.saved_tensors_hooks):
    """Store saved activations compressed while this context is active.

    A saved tensor is compressed when it is a CUDA bf16 tensor produced by an operation (not
    a leaf: weights and inputs are saved as they are), its last dimension N is a multiple of
    group * 8 / bits, it holds at least ``min_numel`` elements, and ``accept(t)`` (if given)
    returns True.  ``basis_for(N)`` may return a LowRankBasis for that width (rank 0 when it
    returns None or is not given).  ``stats`` counts the tensors and bytes compressed.
    """

    def __init__(self, bits: int = 4, group: int = 64,
                 basis_for: Optional[Callable[[int], Optional[LowRankBasis]]] = None,
                 min_numel: int = 1 << 16, accept: Optional[Callable[[torch.Tensor], bool]] = None):
        np_ = 8 // bits
        self.stats = {"compressed": 0, "kept": 0, "bytes_in": 0, "bytes_out": 0}

        def pack(t: torch.Tensor):
            ok = (t.is_cuda and t.dtype == torch.bfloat16 and t.dim() >= 1 and t.grad_fn is not None
                  and t.shape[-1] % (group * np_) == 0 and t.numel() >= min_numel
                  and (accept is None or accept(t)))
            if not ok:
                self.stats["kept"] += 1
                return t
            basis = basis_for(t.shape[-1]) if basis_for is not None else None
            c = encode(t.detach(), basis, bits=bits, group_size=group)
            self.stats["compressed"] += 1
            self.stats["bytes_in"] += 2 * t.numel()
            self.stats["bytes_out"] += c.nbytes()
            return c

        def unpack(c):
            if isinstance(c, CompressedActivation):
                return decode(c)
            return c

        super().__init__(pack, unpack)


def fit_basis(x_sample: torch.Tensor, rank: int) -> LowRankBasis:
    """The top-``rank`` right singular vectors of a sample of rows x_sample[..., N] (fp32 SVD),
    as an orthonormal bf16 V[N, rank] on x_sample's device."""
    xs = _flat(x_sample).to(torch.float32)
    _, _, vh = torch.linalg.svd(xs, full_matrices=False)
    v = vh[:rank].mT.contiguous()
    return LowRankBasis(v.to(torch.bfloat16))
