"""Calls of the C ABI on a tensor's device and torch's current stream."""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

# The same values as torch.cuda.current_device() and torch.cuda.current_stream(i).cuda_stream,
# without the 3 us that building a Stream object takes (a small kernel's own time).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)

DTYPES = {torch.float32: _lib.LNET_F32, torch.bfloat16: _lib.LNET_BF16}


def call(device: torch.device, name: str, *args) -> None:
    """``name(*args, stream)`` with ``device`` current; raises on an error status."""
    index = device.index
    fn = getattr(_lib.load(), name)
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


def pointer(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def require_cuda(what: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA only")


def wants_grad(*tensors: Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def single_backward(fn):
    """``once_differentiable`` for the passes that could be differentiated again
    (``create_graph``), without its cost for all others."""
    once = once_differentiable(fn)

    def backward(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return backward
