"""Residual addition and RMSNorm in one pass, with its gradient and an 8-bit output.

The blocks of ALPHABET normalise inside their own kernels
(``_TightFrameBlock.norm``, src/lnet/pac_tight_frame_models.py:1850-1859); these
functions are that norm for the layers around them: ``h = x + residual`` is
rounded to the inputs' type (it is the stream that the next block reads) and
``y = h / sqrt(mean(h^2) + eps) * weight`` is taken from the stream as stored.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch import Tensor

from . import _lib
from ._launch import DTYPES, call, pointer, require_cuda, single_backward, wants_grad

RMS_NORM_EPS = torch.finfo(torch.float32).eps  # nn.RMSNorm's default for fp32


def _check_norm_args(x: Tensor, weight: Tensor, residual: Tensor | None, eps: float) -> None:
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have shape [..., D], got {tuple(x.shape)}")
    if x.dtype not in DTYPES:
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
    if tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"weight must have shape {(x.shape[-1],)}, got {tuple(weight.shape)}")
    if weight.dtype not in DTYPES:
        raise TypeError(f"weight must be float32 or bfloat16, got {weight.dtype}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape {tuple(x.shape)}, "
                             f"got {tuple(residual.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError(f"residual must be {x.dtype}, got {residual.dtype}")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, x on {x.device}")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")


def _rows(x: Tensor) -> int:
    return x.numel() // x.shape[-1]


def _launch_norm(x: Tensor, weight: Tensor, residual: Tensor | None, eps: float,
                 keep_rstd: bool) -> tuple[Tensor, Tensor | None, Tensor | None]:
    """(y, stream or None without a residual, rstd or None) of contiguous tensors."""
    y = torch.empty_like(x)
    stream = None if residual is None else torch.empty_like(x)
    rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if keep_rstd
            else None)
    call(x.device, "lnet_b200_residual_rms_norm", x.data_ptr(), pointer(residual),
         weight.data_ptr(), DTYPES[x.dtype], DTYPES[weight.dtype], _rows(x), x.shape[-1], eps,
         y.data_ptr(), pointer(stream), pointer(rstd))
    return y, stream, rstd


@lru_cache(maxsize=256)
def _workspace_bytes(dtype: int, rows: int, dim: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().lnet_b200_residual_rms_norm_workspace_size(dtype, rows, dim,
                                                                      ctypes.byref(n)),
               "lnet_b200_residual_rms_norm_workspace_size")
    return int(n.value)


def _launch_norm_backward(stream: Tensor, rstd: Tensor, weight: Tensor, dy: Tensor,
                          dstream: Tensor | None, want_weight: bool
                          ) -> tuple[Tensor, Tensor | None]:
    dx = torch.empty_like(stream)
    dweight = torch.empty_like(weight) if want_weight else None
    code = DTYPES[stream.dtype]
    nbytes = _workspace_bytes(code, _rows(stream), stream.shape[-1]) if want_weight else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=stream.device) if nbytes else None
    call(stream.device, "lnet_b200_residual_rms_norm_backward", stream.data_ptr(),
         rstd.data_ptr(), weight.data_ptr(), dy.data_ptr(), pointer(dstream), code,
         DTYPES[weight.dtype], _rows(stream), stream.shape[-1], dx.data_ptr(), pointer(dweight),
         pointer(ws), nbytes)
    return dx, dweight


class _ResidualRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        xc, wc = x.contiguous(), weight.contiguous()
        rc = None if residual is None else residual.contiguous()
        y, stream, rstd = _launch_norm(xc, wc, rc, eps, True)
        ctx.save_for_backward(xc if stream is None else stream, wc, rstd)
        ctx.set_materialize_grads(False)
        return y, x if stream is None else stream  # without a residual the stream is x itself

    @staticmethod
    @single_backward
    def backward(ctx, dy, dstream):
        stream, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        if dy is None:
            return (dstream if need_x else None, torch.zeros_like(weight) if need_w else None,
                    dstream if need_r else None, None)
        dx, dweight = _launch_norm_backward(
            stream, rstd, weight, dy.contiguous(),
            None if dstream is None else dstream.contiguous(), need_w)
        return dx if need_x else None, dweight, dx if need_r else None, None


def residual_rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None,
                      eps: float = RMS_NORM_EPS) -> tuple[Tensor, Tensor]:
    """``(y, stream)``: ``stream = x + residual`` (``x`` itself without one) and its RMSNorm
    ``y = stream / sqrt(mean(stream^2) + eps) * weight`` over the last dimension.

    ``x`` and ``residual`` [..., D] are float32 or bfloat16 (one type), ``weight`` [D] either.
    Sums and statistics are fp32.  Differentiable in ``x``, ``residual`` and ``weight``.
    """
    _check_norm_args(x, weight, residual, eps)
    require_cuda("residual_rms_norm", x)
    if wants_grad(x, weight, residual):
        return _ResidualRmsNorm.apply(x, weight, residual, eps)
    y, stream, _ = _launch_norm(x.contiguous(), weight.contiguous(),
                                None if residual is None else residual.contiguous(), eps, False)
    return y, x if stream is None else stream


def residual_rms_norm_fp8(x: Tensor, weight: Tensor, residual: Tensor | None = None,
                          eps: float = RMS_NORM_EPS) -> tuple[Tensor, Tensor, Tensor]:
    """``(values, scales, stream)``: the norm of :func:`residual_rms_norm` in 8 bits, for
    :func:`lnet_b200.linear_act_fp8`.

    ``scales`` [...] = max|y| / 448 a row (fp32) and ``values`` [..., D] (``float8_e4m3fn``)
    = y / scale rounded to nearest even; a zero row has scale 0 and values 0.  A serving form:
    it has no gradient and refuses inputs that want one.
    """
    _check_norm_args(x, weight, residual, eps)
    require_cuda("residual_rms_norm_fp8", x)
    if wants_grad(x, weight, residual):
        raise RuntimeError("residual_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    x, weight = x.contiguous(), weight.contiguous()
    residual = None if residual is None else residual.contiguous()
    values = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    stream = None if residual is None else torch.empty_like(x)
    call(x.device, "lnet_b200_residual_rms_norm_fp8", x.data_ptr(), pointer(residual),
         weight.data_ptr(), DTYPES[x.dtype], DTYPES[weight.dtype], _rows(x), x.shape[-1], eps,
         values.data_ptr(), scales.data_ptr(), pointer(stream))
    return values, scales, x if stream is None else stream


__all__ = ["RMS_NORM_EPS", "residual_rms_norm", "residual_rms_norm_fp8"]
