"""Dropout in front of the residual sum, alone and with the LayerNorm that reads the sum next.

The reference trains its pair stack with such updates (protenix/model/modules/fused_ops.py:40-113,
`dropout_add_rowwise`: z + dropout(update), one mask for all rows of the pair tensor).  The mask is never stored: forward
and backward draw it from a counter-based generator (Philox4x32-10, include/protenix_amd.h has the counters), so
that it is a function of the seed and of an element's place in its mask only - the same for every type, layout and
launch, and for a captured call's replays as for the call itself.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import native, ops

Seed = Union[None, int, torch.Tensor]


def _rows(x: torch.Tensor, shared_dim: Optional[int]) -> tuple:
    """(rows, cols, shared, inner): x's rows are [outer][shared][inner]."""
    shape = x.shape
    if not shape:
        raise RuntimeError("x needs at least one dimension")
    cols = shape[-1]
    rows = math.prod(shape[:-1])
    if cols >= (1 << 31) - 8:
        raise RuntimeError(f"rows of {cols} columns: below 2^31 (unsupported shape)")
    if shared_dim is None:
        return rows, cols, 1, 1
    d = shared_dim + len(shape) if shared_dim < 0 else shared_dim
    if not 0 <= d < len(shape) - 1:
        raise RuntimeError(f"shared_dim={shared_dim}: a mask can be shared along any dimension but the last of {tuple(shape)}")
    return rows, cols, max(shape[d], 1), max(math.prod(shape[d + 1:-1]), 1)


def _drawn(x: torch.Tensor) -> int:
    with torch.cuda.device(x.device):
        recorded = torch.cuda.is_current_stream_capturing()
    if recorded:
        raise RuntimeError("a call recorded into a graph needs its seed: every replay would repeat the mask of a seed drawn now "
                           "(give a one-element int64 GPU tensor and change it between replays, or a whole number)")
    return int(torch.empty((), dtype=torch.int64).random_())      # torch's default generator: torch.manual_seed decides


def _seed(seed: Seed, p: float, x: torch.Tensor) -> tuple:
    if p == 0.0:
        return 0, None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise RuntimeError(f"a seed tensor holds one int64 on {x.device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
        return 0, seed
    seed = operator.index(seed)
    if not -(1 << 63) <= seed < 1 << 64:
        raise RuntimeError(f"seed={seed} does not fit 64 bits")
    return seed & 0xFFFFFFFFFFFFFFFF, None


def _check(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, training: bool) -> float:
    ops._dev(x, "x")
    ops._dt_ln(x)
    if residual is not None:
        if residual.device != x.device or residual.shape != x.shape:
            raise RuntimeError(f"x {tuple(x.shape)} on {x.device} and residual {tuple(residual.shape)} on {residual.device} differ")
        if residual.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"a residual is of x's type or float32, got {residual.dtype} beside {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"p={p} is not a probability")
    return p if training else 0.0


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rows, p, number, seed):
        ctx.rows, ctx.p, ctx.number, ctx.x_dtype = rows, p, number, x.dtype
        ctx.save_for_backward(seed)      # (a seed changed in place before the backward pass is noticed)
        return ops.dropout_add(x, residual, x.dtype if residual is None else residual.dtype, rows, p, (number, seed))

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        dx = None
        if ctx.needs_input_grad[0]:
            dx = ops.dropout_add(grad, None, ctx.x_dtype, ctx.rows, ctx.p, (ctx.number, ctx.saved_tensors[0]))
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None, None


def _refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """What the native path asks itself: the operators have no forward-mode derivatives."""
    native.host().refuse_tangents([t for t in tensors if t is not None])


def _refuse_foreign_accumulators(*tensors: Optional[torch.Tensor]) -> None:
    """What the native path asks itself: a gradient recorded into a graph must not reach a leaf that an eager graph holds elsewhere."""
    native.host().refuse_foreign_accumulators([t for t in tensors if t is not None])


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, p: float = 0.1, *, shared_dim: Optional[int] = None,
                training: bool = True, seed: Seed = None) -> torch.Tensor:
    """residual + dropout(x), or dropout(x) without a residual; differentiable in both (backward, once; forward-mode is refused).

    x: float32, bfloat16 or float16, any shape; residual: the same shape, in x's type or float32 (an update of 16 bits onto
    the fp32 residual stream).  The result has the residual's type; the sum is formed in fp32 and rounded once.
    p: the probability with which an element is dropped (to exactly 0, whatever it holds); those that stay are divided by
    1 - p.  p = 0 or training=False: residual + x.
    shared_dim: the dimension along which all elements have the same mask (-3: the rows of a pair tensor, as the
    reference's pair stack has it; -2: its columns); not the last one.
    seed: a whole number of 64 bits, or one int64 in a GPU tensor, read when the kernels run (a graph's replays then have the masks of
    what the tensor holds at the time; it must not change between a call and its backward pass).  None: drawn from torch's default
    generator.  Two calls with the same seed and shape have the same mask."""
    if seed is None and training and p != 0.0 and x.is_cuda:
        seed = _drawn(x)
    if ops.use_native_operators():
        out = native.host().dropout_add(x, residual, p, shared_dim, training, seed)
        if out is not None:
            return out
    p = _check(x, residual, p, training)
    rows = _rows(x, shared_dim)
    number, tensor = _seed(seed, p, x)
    if x.numel() == 0:
        return x + x if residual is None else residual + x      # (nothing to launch; shapes and gradients as torch has them)
    _refuse_tangents(x, residual)
    if _wants_grad(x, residual):
        _refuse_foreign_accumulators(x, residual)
        return _DropoutAdd.apply(x, residual, rows, p, number, tensor)
    return ops.dropout_add(x, residual, x.dtype if residual is None else residual.dtype, rows, p, (number, tensor))


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, rows, p, eps, number, seed):
        ctx.set_materialize_grads(False)
        x, residual, weight, bias = (None if t is None else t.contiguous() for t in (x, residual, weight, bias))
        y, h, stats = ops.dropout_add_layer_norm(x, residual, weight, bias, rows, p, eps, (number, seed), True)
        ctx.rows, ctx.p, ctx.number, ctx.x_dtype = rows, p, number, x.dtype
        ctx.param_dtype = torch.float32 if weight is None and bias is None else (weight if weight is not None else bias).dtype
        # the sum itself where the stream is fp32; else what it is formed from (see ptx_dropout_add_layernorm_bwd)
        keep_h = h.dtype == torch.float32
        ctx.save_for_backward(None if keep_h else x, None if keep_h else residual, h if keep_h else None, stats, weight, seed)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, residual, h, stats, weight, seed = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and dh is None:
            return (None,) * 9
        dy, dh = (None if t is None else t.contiguous() for t in (dy, dh))
        grads = ops.dropout_add_layer_norm_backward(dy, dh, x, residual, h, stats, weight, ctx.param_dtype, ctx.rows, ctx.p,
                                                    (ctx.number, seed), (*need[:4], ctx.x_dtype))
        return (*grads, None, None, None, None, None)


def dropout_add_layer_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                           bias: Optional[torch.Tensor] = None, p: float = 0.0, eps: float = 1e-5, *,
                           shared_dim: Optional[int] = None, training: bool = True,
                           seed: Seed = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(LayerNorm(h), h) with h = residual + dropout(x), in one pass; differentiable in x, residual, weight and bias
    (backward, once; forward-mode is refused).

    x, residual, p, shared_dim, training and seed as in `dropout_add`; the norm is over the last dimension (at most 16384), of
    the fp32 sum before it is rounded to h, and has x's type; h has the residual's.  weight, bias: [x.shape[-1]], of one of the
    three types, the same for both, either may be None; their gradients have their type and are summed in fp32, in a fixed
    order.  p = 0 (the default): the residual sum and norm of a network in use."""
    if seed is None and training and p != 0.0 and x.is_cuda:
        seed = _drawn(x)
    if ops.use_native_operators():
        out = native.host().dropout_add_layer_norm(x, residual, weight, bias, p, eps, shared_dim, training, seed)
        if out is not None:
            return out
    p = _check(x, residual, p, training)
    rows = _rows(x, shared_dim)
    cols = rows[1]
    if cols == 0:
        raise RuntimeError("LayerNorm over an empty dimension")
    params = [t for t in (weight, bias) if t is not None]
    for t in params:
        ops._dt_ln(t)
        if t.shape != (cols,) or t.device != x.device or t.dtype != params[0].dtype:
            raise RuntimeError(f"weight and bias are [{cols}] on {x.device} and of one type, got "
                               + ", ".join(f"{tuple(u.shape)} {u.dtype} on {u.device}" for u in params))
    number, tensor = _seed(seed, p, x)
    _refuse_tangents(x, residual, weight, bias)
    if _wants_grad(x, residual, weight, bias):
        _refuse_foreign_accumulators(x, residual, weight, bias)
        return _DropoutAddLayerNorm.apply(x, residual, weight, bias, rows, p, float(eps), number, tensor)
    x, residual, weight, bias = (None if t is None else t.contiguous() for t in (x, residual, weight, bias))
    return ops.dropout_add_layer_norm(x, residual, weight, bias, rows, p, float(eps), (number, tensor), False)[:2]
