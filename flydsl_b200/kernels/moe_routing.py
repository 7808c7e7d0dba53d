"""The router around ragged expert rows, differentiable (B200).

The launchers of ``topk_gating_softmax_kernel``, ``moe_sorting_kernel`` and ``moe_blockscale_2stage.compile_moe_reduction``
are made for inference.  Here are the same steps as functions with gradients, for rows without padding:

    weights, ids = topk_gating(logits, topk)             # gradient: weights -> logits
    plan = route_rows(ids, num_experts)                  # unit-1 sort and its tables
    xs = moe_permute(x, plan)                            # token rows in expert order;  gradient: sums over a token's rows
    ... grouped_linear(xs, w, plan.offsets) ...
    out = moe_combine(rows, weights, plan)               # out[t] = sum_s weights[t, s] * rows[row of (t, s)]

Sums are fp32 in slot order and rounded once, nothing is atomic, calls only enqueue work on the current stream.  A pair
whose expert id lies outside [0, num_experts) has no row: it adds nothing and its weight's gradient is 0.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ._call import MOST_COLUMNS, MOST_ROWS, in_order, on, once, require_count, require_same_device, require_shape, tracked
from .moe_sorting_kernel import moe_sorting_flydsl

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class RoutedRows(NamedTuple):
    """(token, slot) pairs in expert order.  ``sorted_ids`` int32: (slot << 24) | token of every row, in the first
    ``num_valid_ids[0]`` of them; ``offsets`` int32 [experts + 1]: expert e owns rows offsets[e] .. offsets[e+1]-1;
    ``row_index`` int32 [tokens, topk]: row of a pair, or -1."""
    sorted_ids: torch.Tensor
    num_valid_ids: torch.Tensor
    offsets: torch.Tensor
    row_index: torch.Tensor


def _combine_sizes(rows, weights, plan):
    """(tokens, topk, rows, dim) if the arguments are right, in as few steps as it takes; ``_check_plan`` and the rest say
    what is not."""
    try:
        (sorted_ids, nv, _, row_index), dev, i32 = plan, rows.get_device(), torch.int32
        (count, dim), pairs = rows.shape, weights.shape
        tokens, topk = pairs
        if (rows.is_cuda and rows.dtype in _FLOATS and dim >= 8 and not dim % 8 and row_index.shape == pairs
                and weights.dtype is torch.float32 and min(sorted_ids.numel(), tokens * topk) <= count <= sorted_ids.numel()
                and count <= MOST_ROWS and dim <= MOST_COLUMNS and nv.numel() >= 1
                and sorted_ids.dtype is i32 and nv.dtype is i32 and row_index.dtype is i32
                and dev == weights.get_device() == sorted_ids.get_device() == nv.get_device() == row_index.get_device()
                and rows.is_contiguous() and weights.is_contiguous() and sorted_ids.is_contiguous() and nv.is_contiguous()
                and row_index.is_contiguous()):
            return tokens, topk, count, dim
    except (AttributeError, TypeError, ValueError):
        pass
    return None


def _check_plan(plan: RoutedRows, name: str, t: torch.Tensor, rows: int) -> tuple[int, int]:
    if not isinstance(plan, tuple) or len(plan) != 4:
        raise TypeError("plan must be a RoutedRows (see route_rows)")
    sorted_ids, num_valid_ids, offsets, row_index = plan
    for what, p in (("sorted_ids", sorted_ids), ("num_valid_ids", num_valid_ids), ("row_index", row_index)):
        _lib.require_cuda(f"plan.{what}", p, (torch.int32,))
    require_shape("plan.row_index", row_index, (None, None))
    if sorted_ids.numel() < rows or num_valid_ids.numel() < 1:
        raise ValueError(f"plan.sorted_ids has {sorted_ids.numel()} rows, needs {rows}")
    require_same_device(name, t.device, **{"plan.sorted_ids": sorted_ids, "plan.num_valid_ids": num_valid_ids,
                                           "plan.row_index": row_index})
    return row_index.shape


def _require_rows(name: str, t: torch.Tensor) -> None:
    _lib.require_cuda(name, t, _FLOATS)
    require_shape(name, t, (None, None))
    if t.shape[1] < 8 or t.shape[1] % 8:
        raise ValueError(f"{name} must have a positive multiple of 8 columns, got {t.shape[1]}")
    require_count(f"rows of {name}", t.shape[0])
    require_count(f"columns of {name}", t.shape[1], MOST_COLUMNS)


# ------------------------------------------------------------------------- gate
def _gate(logits, topk, renormalize):
    tokens, experts = logits.shape
    with on(logits.device):
        weights = logits.new_empty((tokens, topk), dtype=torch.float32)
        ids = logits.new_empty((tokens, topk), dtype=torch.int32)
        _lib.check(_lib.load().flymoe_topk_gating_softmax(
            logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], weights.data_ptr(), ids.data_ptr(), None, tokens, experts,
            topk, renormalize, _lib.stream_handle(None)), "topk_gating_softmax")
    return weights, ids


class _TopkGating(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, renormalize):
        weights, ids = _gate(logits, topk, renormalize)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)         # no zeros are made for the ids
        # weights that are a softmax over the picks are all that their gradient needs
        ctx.save_for_backward(weights, ids, *(() if renormalize else (logits,)))
        ctx.logits = logits.shape, logits.dtype, renormalize
        return weights, ids

    @staticmethod
    @once
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None
        weights, ids, *logits = ctx.saved_tensors
        (tokens, experts), dtype, renormalize = ctx.logits
        dweights = in_order(dweights)
        with on(weights.device):
            d = weights.new_empty((tokens, experts), dtype=dtype)
            _lib.check(_lib.load().flymoe_topk_gating_softmax_backward(
                _lib.ptr(logits[0]) if logits else None, _lib.DTYPE_CODE[dtype], weights.data_ptr(), ids.data_ptr(),
                dweights.data_ptr(), d.data_ptr(), tokens, experts, ids.shape[1], renormalize, _lib.stream_handle(None)),
                "topk_gating_softmax_backward")
        return d, None, None


def topk_gating(logits: torch.Tensor, topk: int, *, renormalize: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """logits [tokens, experts] (f32, f16, bf16) -> weights f32 [tokens, topk], ids int32 [tokens, topk].

    Selection and weights are those of ``build_topk_gating_softmax_module``: descending logits, ties to the lower id."""
    _lib.require_cuda("logits", logits, _FLOATS)
    require_shape("logits", logits, (None, None))
    experts = logits.shape[1]
    if not 1 <= experts <= 1024:
        raise ValueError(f"logits must have 1 to 1024 experts, got {experts}")
    if not 1 <= int(topk) <= min(32, experts):
        raise ValueError(f"topk must be in [1, min(32, experts)], got {topk}")
    require_count("tokens", logits.shape[0])
    run = _TopkGating.apply if tracked(logits) else _gate
    return run(logits, int(topk), 1 if renormalize else 0)


# ------------------------------------------------------------------------- plan
def route_rows(topk_ids: torch.Tensor, num_experts: int) -> RoutedRows:
    """topk_ids int32 [tokens, topk] -> the pairs in expert order, pairs of one expert in token order (a stable sort)."""
    _lib.require_cuda("topk_ids", topk_ids, (torch.int32,))
    require_shape("topk_ids", topk_ids, (None, None))
    tokens, topk = topk_ids.shape
    if not 1 <= int(num_experts) <= 1024:
        raise ValueError(f"num_experts must be in [1, 1024], got {num_experts}")
    if not 1 <= topk <= min(255, num_experts):
        raise ValueError(f"topk must be in [1, min(255, num_experts)], got {topk}")
    require_count("tokens", tokens, 2 ** 24 - 1)
    require_count("tokens * topk + num_experts", tokens * topk + num_experts)
    dev, i32 = topk_ids.device, torch.int32
    with on(dev):
        capacity = tokens * topk + num_experts - topk
        sorted_ids, experts = torch.empty((2, capacity), dtype=i32, device=dev).unbind(0)
        nv = torch.empty(2, dtype=i32, device=dev)
        offsets = torch.empty(num_experts + 1, dtype=i32, device=dev)
        row_index = torch.empty((tokens, topk), dtype=i32, device=dev)
        unused = torch.empty(tokens * topk + capacity, dtype=torch.float32, device=dev)      # the sort carries weights along
        moe_sorting_flydsl(topk_ids, unused[: tokens * topk], sorted_ids, unused[tokens * topk:], experts, nv, None,
                           num_experts, 1)
        _lib.check(_lib.load().flymoe_route_tables(sorted_ids.data_ptr(), experts.data_ptr(), nv.data_ptr(),
                                                   row_index.data_ptr(), offsets.data_ptr(), tokens, topk, num_experts,
                                                   tokens * topk, _lib.stream_handle(None)), "route_tables")
    return RoutedRows(sorted_ids[: tokens * topk], nv, offsets, row_index)


# ------------------------------------------------------------------------- rows
def _combine(rows, weights, plan, sizes):
    sorted_ids, num_valid_ids, _, row_index = plan
    with on(rows.device):
        out = rows.new_empty((sizes[0], sizes[3]))
        rc = _lib.load().flymoe_combine_rows(
            rows.data_ptr(), None if weights is None else weights.data_ptr(), out.data_ptr(), sorted_ids.data_ptr(),
            num_valid_ids.data_ptr(), row_index.data_ptr(), *sizes, _lib.DTYPE_CODE[rows.dtype], _lib.stream_handle(None))
    if rc:
        _lib.check(rc, "combine_rows")
    return out


def _permute(x, plan):
    sorted_ids, num_valid_ids, _, row_index = plan
    tokens, topk = row_index.shape
    rows = tokens * topk
    with on(x.device):
        xs = x.new_empty((rows, x.shape[1]))
        _lib.check(_lib.load().flymoe_permute_rows(
            x.data_ptr(), xs.data_ptr(), sorted_ids.data_ptr(), num_valid_ids.data_ptr(), row_index.data_ptr(), tokens,
            topk, rows, x.shape[1] * x.element_size(), _lib.stream_handle(None)), "permute_rows")
    return xs


# A plan goes into a graph as one object, which costs less than four inputs and saved tensors do; what autograd would look at
# is looked at here: whether it was written between the passes.
def _keep_plan(ctx, plan):
    ctx.plan = plan
    ctx.versions = plan[0]._version, plan[1]._version, plan[3]._version


def _kept_plan(ctx):
    plan = ctx.plan
    if ctx.versions != (plan[0]._version, plan[1]._version, plan[3]._version):
        raise RuntimeError("one of the plan's tensors was modified by an inplace operation after the forward pass")
    return plan


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        _keep_plan(ctx, plan)
        return _permute(x, plan)

    @staticmethod
    @once
    def backward(ctx, dxs):
        plan = _kept_plan(ctx)
        with on(dxs.device):
            dxs = in_order(dxs)
        return _combine(dxs, None, plan, (*plan[3].shape, *dxs.shape)), None


def moe_permute(x: torch.Tensor, plan: RoutedRows) -> torch.Tensor:
    """x [tokens, dim] -> [tokens * topk, dim], row r the token of sorted row r; rows without a pair are zero."""
    _require_rows("x", x)
    tokens, topk = _check_plan(plan, "x", x, 0)
    if x.shape[0] != tokens or plan[0].numel() < tokens * topk:
        raise ValueError(f"x has {x.shape[0]} rows, the plan is for {tokens} tokens of {topk} pairs")
    return _Permute.apply(x, plan) if tracked(x) else _permute(x, plan)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan, sizes):
        ctx.save_for_backward(rows, weights)
        _keep_plan(ctx, plan)
        ctx.sizes = sizes
        return _combine(rows, weights, plan, sizes)

    @staticmethod
    @once
    def backward(ctx, dout):
        rows, weights = ctx.saved_tensors
        sorted_ids, num_valid_ids, _, row_index = _kept_plan(ctx)
        need_rows, need_weights, _, _ = ctx.needs_input_grad
        drows = dw = None
        with on(rows.device):
            dout = in_order(dout)
            if need_rows:
                drows = torch.empty_like(rows)
            if need_weights:
                dw = torch.empty_like(weights)
            rc = _lib.load().flymoe_combine_rows_backward(
                dout.data_ptr(), rows.data_ptr(), weights.data_ptr(), drows.data_ptr() if need_rows else None,
                dw.data_ptr() if need_weights else None, sorted_ids.data_ptr(), num_valid_ids.data_ptr(),
                row_index.data_ptr(), *ctx.sizes, _lib.DTYPE_CODE[rows.dtype], _lib.stream_handle(None))
        if rc:
            _lib.check(rc, "combine_rows_backward")
        return drows, dw, None, None


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, plan: RoutedRows) -> torch.Tensor:
    """rows [tokens * topk, dim] in expert order, weights f32 [tokens, topk] -> [tokens, dim]; gradients reach rows and
    weights.  A plan whose ``sorted_ids`` are cut off behind its last pair takes as many rows as it then names, a longer one up to
    as many as it has."""
    sizes = _combine_sizes(rows, weights, plan)
    if sizes is None:
        _require_rows("rows", rows)
        tokens, topk = _check_plan(plan, "rows", rows, rows.shape[0])
        _lib.require_cuda("weights", weights, (torch.float32,))
        require_shape("weights", weights, (tokens, topk))
        if rows.shape[0] < min(plan[0].numel(), tokens * topk):
            raise ValueError(f"rows has {rows.shape[0]} rows, the plan is for {min(plan[0].numel(), tokens * topk)}")
        require_same_device("rows", rows.device, weights=weights)
        sizes = tokens, topk, *rows.shape
    if tracked(rows, weights):
        return _Combine.apply(rows, weights, plan, sizes)
    return _combine(rows, weights, plan, sizes)
