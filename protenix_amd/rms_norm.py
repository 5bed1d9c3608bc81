"""The residual sum and its root-mean-square norm, in x's type or in the 8-bit blocks that `matmul_fp8` reads next."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import native, ops
from .dropout import _refuse_foreign_accumulators, _refuse_tangents, _wants_grad
from .fp8 import Fp8Tensor


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        given = x
        x, residual, weight = (None if t is None else t.contiguous() for t in (x, residual, weight))
        y, h, rstd = ops.add_rms_norm(x, residual, weight, eps, False, True)
        ctx.x_dtype = x.dtype
        # the sum itself where the stream is fp32 (x without a residual); else what it is formed from (see ptx_add_rms_norm_bwd)
        stream = x if h is None else h
        wide = stream.dtype == torch.float32
        ctx.save_for_backward(None if wide else x, None if wide else residual, stream if wide else None, rstd, weight)
        # (without a residual x comes back as a second result, so that its gradient is added before the rounding)
        return y, given if h is None else h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, residual, h, rstd, weight = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 4
        dy, dh = (None if t is None else t.contiguous() for t in (dy, dh))
        return (*ops.add_rms_norm_backward(dy, dh, x, residual, h, rstd, weight, ctx.x_dtype, ctx.needs_input_grad[:3]), None)


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
                 quantize: bool = False) -> Tuple[Union[torch.Tensor, Fp8Tensor], torch.Tensor]:
    """(y, h) with h = residual + x and y = h / sqrt(mean(h^2) + eps) * weight over the last dimension (at most 16384), in one pass;
    differentiable in x, residual and weight (backward, once; forward-mode is refused).

    x: float32, bfloat16 or float16, any shape; residual: the same shape, in x's type or float32; without one h is x itself.  The
    norm is of the fp32 sum before it is rounded to h.  y has x's type, h the residual's.  weight: [x.shape[-1]], of one of the three
    types, or None; its gradient is summed in fp32, in a fixed order.
    quantize: y as an `Fp8Tensor`, blocks along the last dimension, straight from the fp32 values, for `matmul_fp8` and `linear_fp8`
    in use (no gradients)."""
    if ops.use_native_operators():
        out = native.host().add_rms_norm(x, residual, weight, eps, quantize)
        if out is not None:
            return (Fp8Tensor._of(out[0], x.shape), out[1]) if quantize else out
    ops._dev(x, "x")
    ops._dt_ln(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError(f"a norm over the last dimension of {tuple(x.shape)}")
    if x.shape[-1] > 16384:      # (here, since a column count travels in 32 bits)
        raise RuntimeError(f"a norm over at most 16384 columns, got {x.shape[-1]}")
    if residual is not None:
        if residual.device != x.device or residual.shape != x.shape:
            raise RuntimeError(f"x {tuple(x.shape)} on {x.device} and residual {tuple(residual.shape)} on {residual.device} differ")
        if residual.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"a residual is of x's type or float32, got {residual.dtype} beside {x.dtype}")
    if weight is not None:
        ops._dt_ln(weight)
        if weight.shape != x.shape[-1:] or weight.device != x.device:
            raise RuntimeError(f"the weight is [{x.shape[-1]}] on {x.device}, got {tuple(weight.shape)} on {weight.device}")
    _refuse_tangents(x, residual, weight)
    if _wants_grad(x, residual, weight):
        if quantize:
            raise RuntimeError("a norm in 8 bits has no gradients: call under torch.no_grad(), or let linear_fp8 quantize the norm")
        _refuse_foreign_accumulators(x, residual, weight)
        return _AddRMSNorm.apply(x, residual, weight, float(eps))
    shape, given = x.shape, x
    x, residual, weight = (None if t is None else t.contiguous() for t in (x, residual, weight))
    y, h, _ = ops.add_rms_norm(x, residual, weight, float(eps), bool(quantize), False)
    return Fp8Tensor._of(y, shape) if quantize else y, given if h is None else h
