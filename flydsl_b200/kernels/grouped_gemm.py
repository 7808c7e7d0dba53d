"""Matrix products grouped by expert over ragged, unpadded rows, with both gradients (B200, bf16 / fp16).

``moe_gemm_2stage`` multiplies rows that the sort padded to row blocks and is made for inference.  The functions here take
the rows of a unit-1 sort (``moe_routing.route_rows``) or any other ragged batch -- expert ``e`` owns rows
``offsets[e] .. offsets[e+1]-1`` -- and exist in the three forms that training needs:

* ``grouped_gemm(x, w, offsets)``         ``y[r]  = x[r] . w[e(r)]^T``       [rows, k], [experts, n, k] -> [rows, n]
* ``grouped_gemm_dgrad(dy, w, offsets)``  ``dx[r] = dy[r] . w[e(r)]``        [rows, n], [experts, n, k] -> [rows, k]
* ``grouped_gemm_wgrad(dy, x, offsets)``  ``dw[e] = sum_r dy[r]^T x[r]``     [rows, n], [rows, k] -> [experts, n, k]
* ``grouped_linear(x, w, offsets)``       ``grouped_gemm`` with its gradients in autograd

Products are summed in fp32 and rounded once.  ``offsets`` is an int32 tensor [experts + 1] on the GPU and is never read on
the host, so a call only enqueues work.  It has to ascend within [0, rows]; what does not is taken into that range.
Experts may have no rows (``dw[e]`` is then zero).  Rows in front of the first segment and behind the last belong to no
expert: they are zero in a result that the call allocates, and left as they were in the caller's ``out``.

``n`` and ``k`` are multiples of 8, ``experts`` at most 1024, tensors contiguous.  The reference has no gradients and no
unpadded form (its grouped GEMMs: kernels/moe_gemm_2stage.py:90-108, :1780-1796).
"""

from __future__ import annotations

import torch

from .. import _lib
from ._call import HALF, MOST_COLUMNS, MOST_ROWS, in_order, on, once, require_apart, require_count, require_same_device, \
    require_shape, tracked


def _check(rows_name, rows, mats_name, mats, offsets, out, out_shape):
    _lib.require_cuda(rows_name, rows, HALF)
    _lib.require_cuda(mats_name, mats, (rows.dtype,))
    _lib.require_cuda("offsets", offsets, (torch.int32,))
    if out is not None:
        _lib.require_cuda("out", out, (rows.dtype,))
        require_shape("out", out, out_shape)
        require_apart(out, **{rows_name: rows, mats_name: mats})
    require_same_device(rows_name, rows.device, **{mats_name: mats, "offsets": offsets, "out": out})


def _check_sizes(rows, experts, n, k):
    if not 1 <= experts <= 1024:
        raise ValueError(f"experts must be in [1, 1024], got {experts}")
    if n < 8 or n % 8 or k < 8 or k % 8:
        raise ValueError(f"n ({n}) and k ({k}) must be positive multiples of 8")
    require_count("rows", rows)
    require_count("n and k", max(n, k), MOST_COLUMNS)


def _sizes(t, w, offsets, out, input_grad):
    """(rows, experts, n, k) if the arguments are right, in as few steps as it takes; ``_check_rows_form`` says what is not."""
    try:
        (experts, n, k), (rows, inner), (bounds,), dt = w.shape, t.shape, offsets.shape, t.dtype
        if (t.is_cuda and dt in HALF and inner == (n if input_grad else k) and bounds == experts + 1 and w.dtype is dt
                and offsets.dtype is torch.int32 and t.get_device() == w.get_device() == offsets.get_device()
                and t.is_contiguous() and w.is_contiguous() and offsets.is_contiguous() and n >= 8 and not n % 8 and k >= 8
                and not k % 8 and 1 <= experts <= 1024 and rows <= MOST_ROWS and n <= MOST_COLUMNS and k <= MOST_COLUMNS
                and out is None):
            return rows, experts, n, k
    except (AttributeError, ValueError):
        pass
    return None


def _check_rows_form(name, t, w, offsets, out, input_grad):
    if not (isinstance(t, torch.Tensor) and isinstance(w, torch.Tensor) and isinstance(offsets, torch.Tensor)):
        raise TypeError(f"{name}, w and offsets must be torch.Tensors")
    require_shape("w", w, (None, None, None))
    experts, n, k = w.shape
    _check_sizes(t.shape[0] if t.dim() else 0, experts, n, k)
    require_shape(name, t, (None, n if input_grad else k))
    require_shape("offsets", offsets, (experts + 1,))
    _check(name, t, "w", w, offsets, out, (t.shape[0], k if input_grad else n))
    return t.shape[0], experts, n, k


def _rows_form(name, t, w, offsets, out, stream, input_grad):
    sizes = _sizes(t, w, offsets, out, input_grad) or _check_rows_form(name, t, w, offsets, out, input_grad)
    return _run_rows_form(t, w, offsets, out, stream, input_grad, sizes)


def _run_rows_form(t, w, offsets, out, stream, input_grad, sizes):
    with on(t.device, stream):
        res = t.new_empty((sizes[0], sizes[3 if input_grad else 2])) if out is None else out
        rc = _lib.load().flymoe_grouped_gemm(
            res.data_ptr(), t.data_ptr(), w.data_ptr(), offsets.data_ptr(), *sizes, _lib.DTYPE_CODE[t.dtype],
            1 if input_grad else 0, 1 if out is None else 0, _lib.stream_handle(None))
    if rc:
        _lib.check(rc, "grouped_gemm")
    return res


def grouped_gemm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, out: torch.Tensor | None = None, stream=None):
    """x [rows, k], w [experts, n, k], offsets int32 [experts + 1] -> [rows, n]."""
    return _rows_form("x", x, w, offsets, out, stream, False)


def grouped_gemm_dgrad(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, out: torch.Tensor | None = None,
                       stream=None):
    """dy [rows, n], w [experts, n, k] -> the gradient of ``grouped_gemm`` with respect to its rows, [rows, k]."""
    return _rows_form("dy", dy, w, offsets, out, stream, True)


def grouped_gemm_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, *, out: torch.Tensor | None = None,
                       stream=None):
    """dy [rows, n], x [rows, k] -> the gradient of ``grouped_gemm`` with respect to its weights, [experts, n, k]."""
    if not (isinstance(dy, torch.Tensor) and isinstance(x, torch.Tensor) and isinstance(offsets, torch.Tensor)):
        raise TypeError("dy, x and offsets must be torch.Tensors")
    require_shape("dy", dy, (None, None))
    rows, n = dy.shape
    require_shape("x", x, (rows, None))
    k = x.shape[1]
    require_shape("offsets", offsets, (None,))
    experts = offsets.shape[0] - 1
    _check_sizes(rows, experts, n, k)
    _check("dy", dy, "x", x, offsets, out, (experts, n, k))
    with on(dy.device, stream):
        return _wgrad(dy, x, offsets, dy.new_empty((experts, n, k)) if out is None else out)


def _wgrad(dy, x, offsets, out):
    experts, n, k = out.shape
    _lib.check(_lib.load().flymoe_grouped_gemm_wgrad(out.data_ptr(), dy.data_ptr(), x.data_ptr(), offsets.data_ptr(),
                                                     x.shape[0], experts, n, k, _lib.DTYPE_CODE[dy.dtype],
                                                     _lib.stream_handle(None)), "grouped_gemm_wgrad")
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, sizes):
        ctx.save_for_backward(x, w, offsets)
        ctx.sizes = sizes
        return _run_rows_form(x, w, offsets, None, None, False, sizes)

    @staticmethod
    @once
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dy = in_order(dy)
        dx = _run_rows_form(dy, w, offsets, None, None, True, ctx.sizes) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            with on(x.device):
                dw = _wgrad(dy, x, offsets, torch.empty_like(w))
        return dx, dw, None, None


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``grouped_gemm`` in autograd: gradients reach ``x`` and ``w``.  Runs on the current stream."""
    sizes = _sizes(x, w, offsets, None, False) or _check_rows_form("x", x, w, offsets, None, False)
    if tracked(x, w):
        return _GroupedLinear.apply(x, w, offsets, sizes)
    return _run_rows_form(x, w, offsets, None, None, False, sizes)
