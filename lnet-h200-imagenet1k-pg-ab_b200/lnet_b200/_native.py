"""The host path of the feed-forward and distillation operators (``csrc/torch_ops.cpp``): a CPython
module over the C ABI that allocates outputs, launches on torch's current stream and records
gradients.  Built in-tree by :mod:`lnet_b200.build` and loaded on first use; there is no fallback, and a
module of other sources is not loaded.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading

import torch
from torch import Tensor

from . import _lib
from . import build as _build

DTYPES = (torch.float32, torch.bfloat16)

_lock = threading.Lock()
_module = None


def native():
    """The loaded module, bound to the library that :func:`lnet_b200._lib.load` loaded."""
    return _module if _module is not None else _load()


def _load():
    global _module
    with _lock:
        if _module is not None:
            return _module
        lib = _lib.load()
        path = _build.build_torch_ops()
        loader = importlib.machinery.ExtensionFileLoader("_torch_ops", str(path))
        spec = importlib.util.spec_from_file_location("_torch_ops", str(path), loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
                      for name in module.entries()))
        _module = module
        return module


def require_cuda(what: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA only")


def refuse_grad(what: str, *tensors: Tensor | None) -> None:
    """The serving forms have no gradient; silence would cut the graph."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
