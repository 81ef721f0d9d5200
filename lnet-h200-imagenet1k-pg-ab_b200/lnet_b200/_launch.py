"""Calls of the C ABI on a tensor's device and torch's current stream."""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib

DTYPES = {torch.float32: _lib.LNET_F32, torch.bfloat16: _lib.LNET_BF16}


def call(device: torch.device, name: str, *args) -> None:
    """``name(*args, stream)`` with ``device`` current; raises on an error status."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == device.index:
        status = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch.cuda.current_stream().cuda_stream)
    if status:
        _lib.check(status, name)


def pointer(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def require_cuda(what: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA only")


def wants_grad(*tensors: Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
