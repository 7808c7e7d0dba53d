"""Low-rank adapters of many requests at once, beside a shared projection (B200, bf16 / fp16).

``lora_add(y, x, a, b, adapter_ids, scaling)`` adds every row's own adapter to the output of a projection that all rows
share (``compile_blockscale_preshuffle_gemm`` or any other):

    out[m] = y[m] + scaling[l] * b[l] (a[l] x[m]),   l = adapter_ids[m]

    y [rows, n], x [rows, k], a [adapters, rank, k], b [adapters, n, rank]    bf16 or fp16, all of one type, contiguous
    adapter_ids int32 [rows]   any order, one request a row or runs of rows; an id outside [0, adapters) means no adapter
    scaling     f32 [adapters]

The product with ``a`` is summed in fp32 and enters the second one with 16 (bf16) or 22 (fp16) significant bits; the result
is rounded once.  ``out=`` takes the caller's buffer and may be ``y`` itself (serving: in place).  Gradients reach y, x, a
and b; adapters of smaller rank are padded with zeros by the caller.  rank is a multiple of 8 up to 128, k and n multiples of
8.  A row's result depends on its own inputs and adapter only; nothing is atomic.  The reference has no counterpart.
"""

from __future__ import annotations

import torch

from .. import _lib
from ._call import HALF, MOST_COLUMNS, MOST_ROWS, in_order, on, once, require_apart, require_count, require_same_device, \
    require_shape, tracked

MAX_RANK = 128


def _fits(y, x, a, b, ids, scaling, out):
    """Whether the arguments are right, in as few steps as it takes; ``_check`` says what is not."""
    try:
        (rows, k), (adapters, rank, ka), n, dt = x.shape, a.shape, y.shape[1], x.dtype
        return (x.is_cuda and dt in HALF and ka == k and y.shape == (rows, n) and b.shape == (adapters, n, rank)
                and ids.shape == (rows,) and scaling.shape == (adapters,) and y.dtype is dt and a.dtype is dt and b.dtype is dt
                and ids.dtype is torch.int32 and scaling.dtype is torch.float32 and x.get_device() == y.get_device()
                == a.get_device() == b.get_device() == ids.get_device() == scaling.get_device() and x.is_contiguous()
                and y.is_contiguous() and a.is_contiguous() and b.is_contiguous() and ids.is_contiguous()
                and scaling.is_contiguous() and 8 <= rank <= MAX_RANK and not rank % 8 and k >= 8 and not k % 8 and n >= 8
                and not n % 8 and 1 <= adapters <= 32767 and rows <= MOST_ROWS and k <= MOST_COLUMNS and n <= MOST_COLUMNS
                and out is None)
    except (AttributeError, ValueError, IndexError):
        return False


def _check(y, x, a, b, adapter_ids, scaling, out):
    for name, t in (("y", y), ("x", x), ("a", a), ("b", b), ("adapter_ids", adapter_ids), ("scaling", scaling)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    require_shape("x", x, (None, None))
    rows, k = x.shape
    require_shape("a", a, (None, None, k))
    adapters, rank, _ = a.shape
    require_shape("y", y, (rows, None))
    n = y.shape[1]
    require_shape("b", b, (adapters, n, rank))
    require_shape("adapter_ids", adapter_ids, (rows,))
    require_shape("scaling", scaling, (adapters,))
    if rank < 8 or rank % 8 or rank > MAX_RANK:
        raise ValueError(f"rank must be a multiple of 8 in [8, {MAX_RANK}], got {rank}")
    if k < 8 or k % 8 or n < 8 or n % 8:
        raise ValueError(f"k ({k}) and n ({n}) must be positive multiples of 8")
    if not 1 <= adapters <= 32767:
        raise ValueError(f"adapters must be in [1, 32767], got {adapters}")
    require_count("rows", rows)
    require_count("k and n", max(k, n), MOST_COLUMNS)
    _lib.require_cuda("x", x, HALF)
    for name, t in (("y", y), ("a", a), ("b", b), ("out", out)):
        if t is not None:
            _lib.require_cuda(name, t, (x.dtype,))
    if out is not None:
        require_shape("out", out, (rows, n))
        require_apart(out, x=x, a=a, b=b)
        if out.data_ptr() != y.data_ptr():
            require_apart(out, y=y)
    _lib.require_cuda("adapter_ids", adapter_ids, (torch.int32,))
    _lib.require_cuda("scaling", scaling, (torch.float32,))
    require_same_device("x", x.device, y=y, a=a, b=b, adapter_ids=adapter_ids, scaling=scaling, out=out)


def _add(out, y, x, a, b, ids, scaling, keep_v):
    """Enqueues the forward pass; returns v (in the first numbers of a tensor) if ``keep_v``."""
    lib, (rows, k), (adapters, rank, _) = _lib.load(), x.shape, a.shape
    elems = lib.flymoe_lora_v_elems(rows, k, rank)
    v = x.new_empty(elems, dtype=torch.float32)
    kept = None
    if keep_v:                                   # sums in several pieces are scratch, which is not kept alive for one
        kept = v if elems < 2 * rows * rank else x.new_empty(rows * rank, dtype=torch.float32)
    _lib.check(lib.flymoe_lora_forward(out.data_ptr(), y.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(),
                                       scaling.data_ptr(), _lib.ptr(kept), v.data_ptr(), elems, rows, k, y.shape[1], rank,
                                       adapters, _lib.DTYPE_CODE[x.dtype], _lib.stream_handle(None)), "lora_add")
    return kept


class _LoraAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, ids, scaling):
        with on(x.device):
            out = torch.empty_like(y)
            v = _add(out, y, x, a, b, ids, scaling, ctx.needs_input_grad[3])       # only the gradient of b wants it
        ctx.save_for_backward(x, a, b, ids, scaling, v)
        return out

    @staticmethod
    @once
    def backward(ctx, dout):
        x, a, b, ids, scaling, v = ctx.saved_tensors
        need_y, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        dx = da = db = None
        if need_x or need_a or need_b:
            lib, (rows, k), (adapters, n, rank) = _lib.load(), x.shape, b.shape
            with on(x.device):
                dout = in_order(dout)
                elems = lib.flymoe_lora_backward_workspace_elems(rows, k, n, rank, adapters)
                work = x.new_empty(elems, dtype=torch.float32)
                if need_x:
                    dx = torch.empty_like(x)
                if need_a:
                    da = torch.empty_like(a)
                if need_b:
                    db = torch.empty_like(b)
                _lib.check(lib.flymoe_lora_backward(
                    _lib.ptr(dx), _lib.ptr(da), _lib.ptr(db), dout.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(),
                    ids.data_ptr(), scaling.data_ptr(), _lib.ptr(v), work.data_ptr(), elems, rows, k, n, rank, adapters,
                    _lib.DTYPE_CODE[x.dtype], _lib.stream_handle(None)), "lora_backward")
        return dout if need_y else None, dx, da, db, None, None


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor,
             scaling: torch.Tensor, *, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """y + scaling[l] * (x a[l]^T) b[l]^T with l = adapter_ids of the row; see the module docstring.

    With ``out`` or ``stream`` the call is for inference only (no input may require a gradient while gradients are on)."""
    if not _fits(y, x, a, b, adapter_ids, scaling, out):
        _check(y, x, a, b, adapter_ids, scaling, out)
    if tracked(y, x, a, b, scaling):
        if scaling.requires_grad:
            raise ValueError("scaling has no gradient here: detach it, or put it into b")
        if out is not None or stream is not None:
            raise ValueError("out= and stream= are for inference: an input requires a gradient or has a tangent")
        return _LoraAdd.apply(y, x, a, b, adapter_ids, scaling)
    with on(x.device, stream):
        if out is None:
            out = torch.empty_like(y)
        _add(out, y, x, a, b, adapter_ids, scaling, False)
    return out
