"""A learned bias per head and bucket of relative position: `Bias2` of the attention operator where it comes from the tokens'
places in their chains instead of a pair tensor.

    bias[b, h, i, j] = table[bucket(key_positions[b, j] - query_positions[b, i]), h]

`tri_attention(q, k, v, [mask_bias, bias])` takes it as it is ([*, H, Q, K]); the operator's gradient for it comes back as
the table's.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, native, ops
from .dropout import _refuse_foreign_accumulators, _refuse_tangents, _wants_grad

Positions = Union[range, torch.Tensor]
MAX_BUCKETS, MAX_DISTANCE = 255, 8192      # as the kernels take them


class RelativeBuckets:
    """Which bucket a relative position d = key - query falls into.

    num_buckets=None: one bucket per distance up to max_distance, farther ones with the last: max_distance + clip(d, -max_distance,
    max_distance) of 2 max_distance + 1 buckets (residue offsets as the reference's relative position encoding clips them),
    or clip(-d, 0, max_distance) of max_distance + 1 where not bidirectional.
    num_buckets given: a side's first half of its buckets hold one distance each, e of them, the others widen up to max_distance:
    bucket e + j begins at the first n with (n / e)^s >= (max_distance / e)^j, s of them, the last one without an end (found
    in whole numbers, so that a distance at a border is in the bucket the formula says).  A bidirectional scheme has the keys behind the
    query (d > 0) in the upper half of the buckets; else d > 0 counts as 0."""

    def __init__(self, max_distance: int, num_buckets: Optional[int] = None, *, bidirectional: bool = True) -> None:
        max_distance = int(max_distance)
        if not 1 <= max_distance <= MAX_DISTANCE:
            raise ValueError(f"max_distance={max_distance} outside 1..{MAX_DISTANCE}")
        s = _lib.RelativeBucketsStruct()
        s.max_distance = max_distance
        if num_buckets is None:
            num_buckets = 2 * max_distance + 1 if bidirectional else max_distance + 1
            if num_buckets > MAX_BUCKETS:
                raise ValueError(f"{num_buckets} buckets, one per distance, are more than {MAX_BUCKETS}: give num_buckets")
            starts = list(range(max_distance + 1))
            if bidirectional:
                s.neg_base, s.neg_step, s.pos_base, s.pos_step = max_distance, -1, max_distance, 1
            else:
                s.neg_base, s.neg_step, s.pos_base, s.pos_step = 0, 1, 0, 0
        else:
            num_buckets = int(num_buckets)
            side = num_buckets // 2 if bidirectional else num_buckets
            exact = side // 2
            if num_buckets > MAX_BUCKETS or side < 2 or (bidirectional and num_buckets % 2):
                raise ValueError(f"num_buckets={num_buckets}: at most {MAX_BUCKETS}, at least 2 a side, an even number of them for two sides")
            if max_distance <= exact:
                raise ValueError(f"max_distance={max_distance} has to exceed the {exact} distances with a bucket of their own")
            starts = list(range(exact)) + _widening(exact, side - exact, max_distance)
            s.neg_base, s.neg_step = 0, 1
            s.pos_base, s.pos_step = (side, 1) if bidirectional else (0, 0)
        s.count, s.side = num_buckets, len(starts)
        s.starts[:len(starts)] = starts
        self._struct = s
        self.max_distance, self.num_buckets, self.bidirectional = max_distance, num_buckets, bool(bidirectional)

    def bucket(self, d: int) -> int:
        """The bucket of one difference key - query."""
        s, n = self._struct, min(abs(d), self.max_distance)
        side = max(j for j in range(s.side) if s.starts[j] <= n)
        return s.pos_base + s.pos_step * side if d > 0 else s.neg_base + s.neg_step * side

    def __repr__(self) -> str:
        return f"RelativeBuckets(max_distance={self.max_distance}, num_buckets={self.num_buckets}, bidirectional={self.bidirectional})"


def _widening(exact: int, count: int, max_distance: int) -> list:
    """The first distance of each of `count` buckets behind `exact` single ones: the smallest n with
    n^count >= max_distance^j exact^(count - j)."""
    starts = []
    for j in range(count):
        bound, lo, hi = max_distance**j * exact ** (count - j), exact, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid**count >= bound:
                hi = mid
            else:
                lo = mid + 1
        starts.append(lo)
    return starts


def _axis(p: Positions, name: str, device: torch.device) -> Tuple[Optional[torch.Tensor], int, int, Optional[int]]:
    """(positions or None, the first one of a range, length, batch size or None)"""
    if isinstance(p, range):
        if p.step != 1:
            raise RuntimeError(f"{name}: a range of positions has step 1, got {p}")
        if not -(1 << 62) <= p.start < 1 << 62:
            raise RuntimeError(f"{name}: positions from {p.start} on")
        return None, p.start, max(p.stop - p.start, 0), None      # (its len() stops at 63 bits)
    return _whole(p, name, device), 0, p.shape[-1], p.shape[0] if p.dim() == 2 else None


def _whole(t: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32) or t.dim() not in (1, 2):
        got = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise RuntimeError(f"{name}: whole numbers [n] or [batch, n] (int64 or int32), got {got}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the table on {device}")
    return t.to(torch.int64)


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, size, batched, q, k, gq, gk, q_first, k_first, dtype):
        ctx.buckets, ctx.size, ctx.first = buckets, size, (q_first, k_first)
        ctx.table_shape, ctx.table_dtype = tuple(table.shape), table.dtype
        ctx.save_for_backward(q, k, gq, gk)
        return ops.relative_bias(buckets._struct, table.contiguous(), size, (q, q_first), (k, k_first), (gq, gk), dtype, batched)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, gq, gk = ctx.saved_tensors
        dtable = ops.relative_bias_backward(ctx.buckets._struct, grad, ctx.table_shape, ctx.table_dtype, ctx.size, (q, ctx.first[0]),
                                            (k, ctx.first[1]), (gq, gk))
        return (dtable,) + (None,) * 10


def relative_position_bias(table: torch.Tensor, buckets: RelativeBuckets, query_positions: Positions, key_positions: Positions, *,
                           groups: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                           dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """[H, Q, K], or [B, H, Q, K] where any of the positions or groups is [B, n]; differentiable in the table (backward, once;
    forward-mode is refused), whose gradient is summed in fp32, in a fixed order.

    table: [buckets.num_buckets, H], float32, bfloat16 or float16 - with one row more, for pairs of different groups, where groups are
    given.  query_positions, key_positions: a `range` of step 1 (range(n, n + 1): the one query of a token
    behind n others), or whole numbers [n] or [B, n]; they may repeat and need no order.
    groups: (of the queries, of the keys), whole numbers of the positions' shapes: tokens of one chain have one number, since residue
    numbers of two chains say nothing about each other.  dtype: of the result (the table's by default)."""
    if ops.use_native_operators():
        out = native.host().relative_bias(table, ctypes.addressof(buckets._struct), query_positions, key_positions, groups, dtype)
        if out is not None:
            return out
    ops._dev(table, "table")
    ops._dt_ln(table)
    dtype = dtype or table.dtype
    if dtype not in ops._LN_DTYPES:
        raise RuntimeError(f"a bias is float32, bfloat16 or float16, got {dtype}")
    rows = buckets.num_buckets + (groups is not None)
    if table.dim() != 2 or table.shape[0] != rows or table.shape[1] == 0:
        raise RuntimeError(f"the table is [{rows}, heads] for {buckets}{' with groups' if groups is not None else ''}, got {tuple(table.shape)}")
    q, q_first, n_q, b_q = _axis(query_positions, "query_positions", table.device)
    k, k_first, n_k, b_k = _axis(key_positions, "key_positions", table.device)
    gq = gk = None
    sizes = [b_q, b_k]
    if groups is not None:
        gq, gk = (_whole(g, "groups", table.device) for g in groups)
        if gq.shape[-1] != n_q or gk.shape[-1] != n_k:
            raise RuntimeError(f"groups of {gq.shape[-1]} queries and {gk.shape[-1]} keys beside positions of {n_q} and {n_k}")
        sizes += [g.shape[0] if g.dim() == 2 else None for g in (gq, gk)]
    batches = {b for b in sizes if b is not None}
    if len(batches) > 1:
        raise RuntimeError(f"positions and groups of different batch sizes {sorted(batches)}")
    batch = batches.pop() if batches else None
    size = (1 if batch is None else batch, table.shape[1], n_q, n_k)
    if max(size[0], n_q, n_k) > 1 << 30:
        raise RuntimeError(f"a batch of {size[0]} with {n_q} queries and {n_k} keys: 2^30 at most (unsupported shape)")
    q, k, gq, gk = (None if t is None else t.expand(size[0], t.shape[-1]).contiguous() for t in (q, k, gq, gk))
    _refuse_tangents(table)
    if _wants_grad(table):
        _refuse_foreign_accumulators(table)
        return _RelativeBias.apply(table, buckets, size, batch is not None, q, k, gq, gk, q_first, k_first, dtype)
    return ops.relative_bias(buckets._struct, table.contiguous(), size, (q, q_first), (k, k_first), (gq, gk), dtype, batch is not None)


class RelativePositionBias(nn.Module):
    """`relative_position_bias` with its table as the parameter `weight` [buckets (+ 1 where `grouped`), heads]."""

    def __init__(self, heads: int, buckets: RelativeBuckets, *, grouped: bool = False) -> None:
        super().__init__()
        self.buckets, self.grouped = buckets, bool(grouped)
        self.weight = nn.Parameter(torch.zeros(buckets.num_buckets + self.grouped, heads))

    def forward(self, query_positions: Positions, key_positions: Positions,
                groups: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        if self.grouped != (groups is not None):
            raise RuntimeError("groups are given exactly where the module was made with grouped=True")
        return relative_position_bias(self.weight, self.buckets, query_positions, key_positions, groups=groups, dtype=dtype)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[1]} heads, {self.buckets}, grouped={self.grouped}"
