"""Linear layers in 8 bits: matrices as e4m3 values with a scale per block of 128, their product, and `linear_fp8` with its gradients.

Where `Linear` multiplies in bf16 or fp32, these multiply at the 8-bit rate of the matrix cores.  A block is 128 values along the axis
that is summed over (activations, gradients), or 128 x 128 (`square`: weights, whose transpose then has the same numbers); its scale
is its largest magnitude over 448, and a product's sums are fp32 (of 16-bit results: see `matmul_fp8`).  The scheme is written down in include/protenix_amd.h.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import native, ops
from .dropout import _refuse_foreign_accumulators, _refuse_tangents, _wants_grad

BLOCK = 128
_MOST_SUMMED = 1 << 24      # values that a product sums over (ptx_fp8_matmul's k)


class Fp8Tensor:
    """A matrix [*, k] in 8-bit blocks along its last dimension, as `quantize_fp8`, `add_rms_norm(quantize=True)` and this class make it.

    values: float8_e4m3fn [*, k]; scales: float32 [*, ceil(k / 128)], or with square=True [ceil(n / 128), ceil(k / 128)] for values
    [n, k].  `values` and `scales` are views of the operand's own memory, whose layout is the kernels'; what is given here is copied
    into that layout (weights of a checkpoint, say), without a graph: tensors inside one are refused, leaves taken."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, *, square: bool = False) -> None:
        ops._dev(values, "values")
        if values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32 or scales.device != values.device:
            raise RuntimeError(f"values are float8_e4m3fn and scales float32 on their device, got {values.dtype} and {scales.dtype} on "
                               f"{values.device} and {scales.device}")
        if values.dim() < 1 or values.shape[-1] == 0 or (square and values.dim() != 2):
            raise RuntimeError(f"values are [*, k] with k > 0, [n, k] with square scales, got {tuple(values.shape)}")
        *lead, k = values.shape
        want = (-(-lead[0] // BLOCK), -(-k // BLOCK)) if square else (*lead, -(-k // BLOCK))
        if tuple(scales.shape) != want:
            raise RuntimeError(f"values {tuple(values.shape)} have scales {want}{' (square)' if square else ''}, got {tuple(scales.shape)}")
        _refuse_lost_gradients(values, scales)
        values, scales, rows = values.detach(), scales.detach(), math.prod(lead)
        with torch.cuda.device(values.device):
            operand = ops.fp8_buffers(rows, k, bool(square), values.device)
            data = operand[0].view(torch.uint8)
            data[:, :k] = values.reshape(rows, k).view(torch.uint8)
            data[:, k:] = 0
            if square:
                operand[1].copy_(scales)
            else:
                operand[1][:, :rows] = scales.reshape(rows, scales.shape[-1]).t()
        self._operand, self.shape = operand, torch.Size(values.shape)

    @classmethod
    def _of(cls, operand: tuple, shape) -> "Fp8Tensor":
        t = cls.__new__(cls)
        t._operand, t.shape = operand, shape if type(shape) is torch.Size else torch.Size(shape)
        return t

    @property
    def values(self) -> torch.Tensor:
        return native.host().fp8_values(self._operand[0], self.shape)

    @property
    def scales(self) -> torch.Tensor:
        return self._operand[1] if self._operand[4] else native.host().fp8_scales(self._operand[1], self.shape)

    @property
    def square(self) -> bool:
        return self._operand[4]

    @property
    def device(self) -> torch.device:
        return self._operand[0].device

    def __repr__(self) -> str:
        return f"Fp8Tensor({tuple(self.shape)}, {'a scale per 128 x 128' if self.square else 'a scale per 128'}, {self.device})"


Operand = Union[torch.Tensor, Fp8Tensor]


def _matrix(x: torch.Tensor, name: str) -> torch.Tensor:
    ops._dev(x, name)
    ops._dt_ln(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError(f"{name} is [*, k] with k > 0, got {tuple(x.shape)}")
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def quantize_fp8(x: torch.Tensor, *, square: bool = False, along: Union[int, Tuple[int, int]] = -1):
    """x [*, k], float32, bfloat16 or float16, in 8-bit blocks.  No gradient: a rounding has none, and `linear_fp8` has its own.  So an x
    inside a graph, or a dual tensor, is refused; a leaf (a weight to serve) is taken, and gets none from here.

    along=-1: blocks of the last dimension; the result has x's shape.  along=-2: the rows (all other dimensions as one) are the axis
    that will be summed over: the transposed matrix [k, rows], blocks along its rows.  along=(-1, -2): both, from one pass over x.
    square: a scale per 128 x 128, for x [n, k]: a weight, laid out once for serving."""
    if ops.use_native_operators():
        both = along == (-1, -2)
        if both or along == -1 or along == -2:
            out = native.host().quantize_fp8(x, square, along != -2, along != -1)
            if out is not None:
                q, qt = out
                first = None if q is None else Fp8Tensor._of(q, x.shape)
                second = None if qt is None else Fp8Tensor._of(qt, (qt[2], qt[3]))
                return (first, second) if both else second if first is None else first
    matrix = _matrix(x, "x")
    if along not in (-1, -2, (-1, -2)):
        raise RuntimeError(f"along={along}: -1, -2 or (-1, -2)")
    if square and x.dim() != 2:
        raise RuntimeError(f"square blocks are of a matrix [n, k], got {tuple(x.shape)}")
    if along != -1 and matrix.shape[0] == 0:
        raise RuntimeError("along=-2: no rows to sum over")
    _refuse_lost_gradients(x)
    q, qt, _ = ops.fp8_quantize(matrix.detach(), bool(square), along != -2, along != -1)
    got = [Fp8Tensor._of(q, x.shape) if q else None, Fp8Tensor._of(qt, (matrix.shape[1], matrix.shape[0])) if qt else None]
    return tuple(got) if along == (-1, -2) else got[along == -2]


def _check_bias(bias: Optional[torch.Tensor], n: int, device: torch.device) -> None:
    if bias is None:
        return
    ops._dt_ln(bias)
    if bias.shape != (n,) or bias.device != device:
        raise RuntimeError(f"the bias is [{n}] on {device}, got {tuple(bias.shape)} on {bias.device}")


def _out_type(dtype: torch.dtype) -> torch.dtype:
    if dtype not in ops._LN_DTYPES:
        raise RuntimeError(f"a product is float32, bfloat16 or float16, got {dtype}")
    return dtype


def matmul_fp8(a: Fp8Tensor, b: Fp8Tensor, bias: Optional[torch.Tensor] = None, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T + bias, [*, n] of type dtype, for a [*, k] and b [n, k]; sums in fp32, rounded once.  16-bit results: of products that the 8-bit
    matrix instruction has cut at 2^-13 of the largest among 8 neighbouring k, 1.4e-5 of a result on normal data and more where large ones
    cancel; float32 ones are formed in fp32 throughout.

    a has a scale per 128 values; b the same, or square ones (a weight).  bias: [n], float32, bfloat16 or float16."""
    if ops.use_native_operators() and isinstance(a, Fp8Tensor) and isinstance(b, Fp8Tensor) and len(b.shape) == 2:
        out = native.host().matmul_fp8(a._operand, b._operand, bias, dtype, a.shape)
        if out is not None:
            return out
    if not isinstance(a, Fp8Tensor) or not isinstance(b, Fp8Tensor):
        raise RuntimeError(f"matmul_fp8 takes two Fp8Tensors, got {type(a).__name__} and {type(b).__name__}")
    if len(b.shape) != 2 or a.shape[-1] != b.shape[1] or a.device != b.device:
        raise RuntimeError(f"a [*, k] and b [n, k] on one device, got {tuple(a.shape)} and {tuple(b.shape)} on {a.device} and {b.device}")
    if a.square:
        raise RuntimeError("a has a scale per 128 values of a row (square scales are b's)")
    _check_bias(bias, b.shape[0], b.device)
    _refuse_tangents(bias)
    _refuse_wanted(bias)
    bias = None if bias is None else bias.contiguous()
    out = ops.fp8_matmul(a._operand, b._operand, bias, _out_type(dtype))
    return out.view(*a.shape[:-1], b.shape[0])


def _refuse_wanted(*tensors: Optional[torch.Tensor]) -> None:
    if _wants_grad(*tensors):
        raise RuntimeError("operands in 8 bits have no gradients: give linear_fp8 the tensors themselves, or call under torch.no_grad()")


def _refuse_lost_gradients(*tensors: torch.Tensor) -> None:
    """What passes a gradient on to others; a leaf is taken as it stands."""
    _refuse_tangents(*tensors)
    _refuse_wanted(*(t for t in tensors if not t.is_leaf))


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, dtype):
        need = ctx.needs_input_grad
        matrix = x.reshape(-1, x.shape[-1])
        xq, xt, _ = ops.fp8_quantize(matrix, False, True, need[1])
        wq, wt, _ = ops.fp8_quantize(weight, True, True, need[0])
        ctx.x_shape, ctx.types = x.shape, (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        # what the gradients take, in 8 bits: neither x nor the weight is kept
        ctx.saved = [None if t is None else t[2:] for t in (xt, wt)]
        ctx.save_for_backward(*(u for t in (xt, wt) for u in (t[:2] if t else (None, None))))
        return ops.fp8_matmul(xq, wq, None if bias is None else bias.contiguous(), dtype).view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        t = ctx.saved_tensors
        xt, wt = (None if s is None else (t[2 * i], t[2 * i + 1], *s) for i, s in enumerate(ctx.saved))
        need = ctx.needs_input_grad
        q, qt, db = ops.fp8_quantize(dy.reshape(math.prod(ctx.x_shape[:-1]), dy.shape[-1]), False, need[0], need[1], ctx.types[2] if need[2] else None)
        dx = ops.fp8_matmul(q, wt, None, ctx.types[0]).view(ctx.x_shape) if need[0] else None
        dw = ops.fp8_matmul(qt, xt, None, ctx.types[1]) if need[1] else None
        return dx, dw, db, None


def linear_fp8(x: Operand, weight: Operand, bias: Optional[torch.Tensor] = None, *, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T + bias with both in 8-bit blocks: [*, n] for x [*, k], weight [n, k], bias [n]; differentiable (backward, once;
    forward-mode is refused).

    x, weight: float32, bfloat16 or float16 tensors, each of its own type, or `Fp8Tensor`s (in use without gradients: a weight laid out
    once by `quantize_fp8(weight, square=True)`, what `add_rms_norm(quantize=True)` left of x).  dtype: of the result (by
    default x's, or for float32 x under torch.autocast that one's; bfloat16 for x in 8 bits); see `matmul_fp8` for the sums of 16-bit ones.
    Training: x and dy in blocks of 128 along the axis each product sums over, the weight in blocks of 128 x 128; dx = dy W and
    dW = dy^T x are products of such operands too, with the rounding to 8 bits taken as the identity, and db is summed in fp32,
    in a fixed order.  Gradients have their inputs' types.  Neither x nor the weight is kept, only their 8-bit forms.  A product sums
    over at most 2^24 values, and so do gradients: rows of x for the weight's, of the weight for x's."""
    if dtype is None and isinstance(x, torch.Tensor):
        dtype = ops.autocast_compute_dtype(x)      # (as `Linear`: for fp32 x under torch.autocast its type)
    if ops.use_native_operators() and isinstance(x, torch.Tensor):
        out = None
        if isinstance(weight, torch.Tensor):
            out = native.host().linear_fp8(x, weight, bias, dtype)
        elif len(weight.shape) == 2:
            out = native.host().linear_fp8_ready(x, weight._operand, bias, dtype)
        if out is not None:
            return out
    if not isinstance(weight, Fp8Tensor):
        _matrix(weight, "weight")
    if len(weight.shape) != 2:
        raise RuntimeError(f"the weight is [n, k], got {tuple(weight.shape)}")
    n, k = weight.shape
    if not isinstance(x, Fp8Tensor):
        _matrix(x, "x")
    if x.shape[-1] != k or x.device != weight.device:
        raise RuntimeError(f"x [*, k] and weight [n, k] on one device, got {tuple(x.shape)} and {tuple(weight.shape)} on {x.device} and {weight.device}")
    _check_bias(bias, n, weight.device)
    dtype = _out_type(dtype or (torch.bfloat16 if isinstance(x, Fp8Tensor) else x.dtype))
    plain = [t for t in (x, weight, bias) if isinstance(t, torch.Tensor)]
    _refuse_tangents(*plain)
    if isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and _wants_grad(*plain):
        _refuse_foreign_accumulators(*plain)
        # (here, and not in the backward pass: the gradients are products over the rows of x and over those of the weight)
        rows = math.prod(x.shape[:-1])
        if (weight.requires_grad and rows > _MOST_SUMMED) or (x.requires_grad and n > _MOST_SUMMED):
            raise RuntimeError(f"gradients of linear_fp8 sum over at most {_MOST_SUMMED} rows, got {rows} of x and {n} of the weight")
        return _LinearFp8.apply(x, weight, bias, dtype)
    if isinstance(x, Fp8Tensor) or isinstance(weight, Fp8Tensor):
        _refuse_wanted(*plain)
    a = x if isinstance(x, Fp8Tensor) else quantize_fp8(x)
    b = weight if isinstance(weight, Fp8Tensor) else quantize_fp8(weight, square=True)
    return matmul_fp8(a, b, None if bias is None else bias.detach(), dtype=dtype)
