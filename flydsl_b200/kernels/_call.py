"""What the operator functions share: the device and stream of a call, and its argument checks."""

from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib

HALF = (torch.bfloat16, torch.float16)
# The library takes sizes as 32-bit numbers, a larger one would arrive as another; the kernels look up to 1024 rows past the last.
MOST_ROWS = 2 ** 31 - 1 - 1024
MOST_COLUMNS = 2 ** 29
_HERE = contextlib.nullcontext()


def on(device: torch.device, stream=None):
    """Context in which a call allocates and launches: the device of its tensors, and ``stream`` (None: that device's
    current one).  What is allocated inside belongs to that stream; the inputs have to be ready on it, as for every
    launcher."""
    if stream is not None:
        if isinstance(stream, int) or not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(_lib.stream_handle(stream), device=device)
        if device.index is not None and stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
        return torch.cuda.stream(stream)
    if device.index is None or device.index == torch._C._cuda_getDevice():     # current_device() without its wrapper
        return _HERE
    return torch.cuda.device(device)


def tracked(*tensors) -> bool:
    """Whether autograd has to see a call: one of its inputs requires a gradient, or carries a tangent of forward mode (which
    the functions here have not, and then say so)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def in_order(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as autograd hands it over (any strides, any place in memory) as the kernels want it: contiguous, 16-byte
    aligned."""
    grad = grad.contiguous()
    return grad.clone() if grad.data_ptr() % 16 else grad


def once(backward):
    """``once_differentiable`` without its steps (2.5 us of host time a call) where no gradient of the gradient is asked for."""
    checked = once_differentiable(backward)

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)

    return wrapper


def require_shape(name: str, t: torch.Tensor, shape: tuple) -> None:
    """``None`` in ``shape`` stands for any size."""
    if t.dim() != len(shape) or any(s is not None and s != d for s, d in zip(shape, t.shape)):
        want = ", ".join("*" if s is None else str(s) for s in shape)
        raise ValueError(f"{name} must have shape [{want}], got {list(t.shape)}")


def require_count(what: str, count: int, most: int = MOST_ROWS) -> None:
    if count > most:
        raise ValueError(f"{what} must not exceed {most}, got {count}")


def require_apart(out: torch.Tensor, **inputs) -> None:
    """``out`` shares no memory with the inputs, which are read while it is written."""
    at, end = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for name, t in inputs.items():
        if at < t.data_ptr() + t.numel() * t.element_size() and t.data_ptr() < end:
            raise ValueError(f"out must not share memory with {name}")


def require_same_device(first: str, device: torch.device, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, {first} on {device}")
