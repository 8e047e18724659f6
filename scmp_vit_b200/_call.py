"""Calls into the engine library on a tensor's device and current stream."""
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib

DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # enum scmp_dtype

try:  # the stream's handle without a Stream object around it
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # a CPU build of torch
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream
try:  # (the tensors of a call exist, so the device is initialised)
    _current_device = torch._C._cuda_getDevice
except AttributeError:
    _current_device = torch.cuda.current_device


_graph_task = getattr(torch._C, "_current_graph_task_id", None)


def in_backward() -> Optional[bool]:
    """Whether this thread is inside a backward pass; None where torch does not tell."""
    return None if _graph_task is None else _graph_task() >= 0


def call(fn, index: int, *args) -> None:
    """``fn(*args, stream)`` on CUDA device ``index`` and its current stream;
    raises on a non-zero status."""
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        if index < 0:
            raise RuntimeError("runs on the CUDA engine only (no CPU path)")
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status)


def in_dual_level() -> bool:
    """Whether forward-mode derivatives are being taken."""
    return _forward_ad._current_level >= 0


def has_tangent(tensors) -> bool:
    """Whether one of the tensors (or None) is a dual one of forward-mode
    differentiation, which ``requires_grad`` and the grad mode do not show."""
    if not in_dual_level():
        return False
    return any([t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors])


def once_differentiable(backward):
    """``torch.autograd.function.once_differentiable``, entered only where a
    gradient of the gradient is being recorded."""
    recorded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return run


def dtype_code(dtype: torch.dtype, what: str) -> int:
    code = DTYPE.get(dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {dtype}")
    return code
