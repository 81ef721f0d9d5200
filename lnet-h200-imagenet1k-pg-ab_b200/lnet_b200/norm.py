"""Residual addition and RMSNorm in one pass, with its gradient and an 8-bit output.

The blocks of ALPHABET normalise inside their own kernels
(``_TightFrameBlock.norm``, src/lnet/pac_tight_frame_models.py:1850-1859); these
functions are that norm for the layers around them: ``h = x + residual`` is
rounded to the inputs' type (it is the stream that the next block reads) and
``y = h / sqrt(mean(h^2) + eps) * weight`` is taken from the stream as stored.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._native import DTYPES, native, refuse_grad, require_cuda

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


def residual_rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None,
                      eps: float = RMS_NORM_EPS) -> tuple[Tensor, Tensor]:
    """``(y, stream)``: ``stream = x + residual`` (``x`` itself without one) and its RMSNorm
    ``y = stream / sqrt(mean(stream^2) + eps) * weight`` over the last dimension.

    ``x`` and ``residual`` [..., D] are float32 or bfloat16 (one type), ``weight`` [D] either.
    Sums and statistics are fp32.  Differentiable in ``x``, ``residual`` and ``weight``.
    """
    _check_norm_args(x, weight, residual, eps)
    require_cuda("residual_rms_norm", x)
    return native().norm(x, weight, residual, eps)


def residual_rms_norm_fp8(x: Tensor, weight: Tensor, residual: Tensor | None = None,
                          eps: float = RMS_NORM_EPS) -> tuple[Tensor, Tensor, Tensor]:
    """``(values, scales, stream)``: the norm of :func:`residual_rms_norm` in 8 bits, for
    :func:`lnet_b200.linear_act_fp8`.

    ``scales`` [...] = max|y| / 448 a row (fp32) and ``values`` [..., D] (``float8_e4m3fn``)
    = y / scale rounded to nearest even; a zero row has scale 0 and values 0.  The quotient has two
    fp32 roundings, so that a value within 2^-22 of a tie may take the neighbouring code.  A serving
    form: it has no gradient and refuses inputs that want one.
    """
    _check_norm_args(x, weight, residual, eps)
    require_cuda("residual_rms_norm_fp8", x)
    refuse_grad("residual_rms_norm_fp8", x, weight, residual)
    return native().norm_fp8(x, weight, residual, eps)


__all__ = ["RMS_NORM_EPS", "residual_rms_norm", "residual_rms_norm_fp8"]
