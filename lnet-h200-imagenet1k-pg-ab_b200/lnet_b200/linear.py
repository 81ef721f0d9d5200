"""Matrix product with bias, activation and residual in its epilogue.

The reference's channel mixing goes through ``torch.nn.Linear`` (the affine
readout, src/lnet/alphabet.py:49-63); these functions are the layer of a
feed-forward block: ``y = f(x W^T + bias) + residual`` in one kernel on tcgen05,
with its gradient, and its serving form on 8-bit operands
(:func:`lnet_b200.residual_rms_norm_fp8` writes them).
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._native import DTYPES, native, refuse_grad, require_cuda

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _check_linear_args(x, weight, bias, residual, activation, operand) -> None:
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have shape [..., K], got {tuple(x.shape)}")
    if x.dtype != operand:
        raise TypeError(f"x must be {operand}, got {x.dtype}")
    if weight.ndim != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"weight must have shape ['N', {x.shape[-1]}], "
                         f"got {tuple(weight.shape)}")
    if weight.dtype != operand:
        raise TypeError(f"weight must be {operand}, got {weight.dtype}")
    n = weight.shape[0]
    for name, t, shape in (("bias", bias, (n,)), ("residual", residual, (*x.shape[:-1], n))):
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be torch.bfloat16, got {t.dtype}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")


def _check_linear_fp8_args(x, x_scale, weight, weight_scale, bias, residual, activation) -> None:
    _check_linear_args(x, weight, bias, residual, activation, torch.float8_e4m3fn)
    for name, t, shape in (("x_scale", x_scale, tuple(x.shape[:-1])),
                           ("weight_scale", weight_scale, (weight.shape[0],))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def linear_act(x: Tensor, weight: Tensor, bias: Tensor | None = None,
               residual: Tensor | None = None, *, activation: str = "none") -> Tensor:
    """``f(x @ weight.T + bias) + residual`` for bfloat16 ``x`` [..., K] and ``weight`` [N, K].

    ``activation`` is ``"none"``, ``"relu"``, ``"silu"`` or ``"gelu"`` (the erf form).  Sums are
    fp32 and the result is rounded once to bfloat16.  Differentiable in ``x``, ``weight``, ``bias``
    and ``residual``.  Through an activation the forward pass keeps a = x W^T + bias in bfloat16, the
    gradient takes f'(a) from it, and da = dy f'(a) is rounded to bfloat16 as an operand of the products
    for ``x`` and ``weight`` (with GELU their gradients are 2.4e-3 of themselves off, 1.7e-3 is the
    rounding of the result alone); ``bias`` sums the unrounded da.
    """
    _check_linear_args(x, weight, bias, residual, activation, torch.bfloat16)
    require_cuda("linear_act", x)
    return native().linear(x, weight, bias, residual, ACTIVATIONS[activation])


def linear_act_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor,
                   bias: Tensor | None = None, residual: Tensor | None = None, *,
                   activation: str = "none") -> Tensor:
    """:func:`linear_act` on 8-bit operands: ``x`` [..., K] and ``weight`` [N, K] are
    ``float8_e4m3fn`` with the fp32 scales ``x_scale`` [...] and ``weight_scale`` [N] of their rows
    (:func:`lnet_b200.residual_rms_norm_fp8`, :func:`quantize_rows_fp8`); bias, residual and the
    result are bfloat16.  A serving form: it has no gradient and refuses inputs that want one.
    """
    _check_linear_fp8_args(x, x_scale, weight, weight_scale, bias, residual, activation)
    require_cuda("linear_act_fp8", x)
    refuse_grad("linear_act_fp8", x, x_scale, weight, weight_scale, bias, residual)
    return native().linear_fp8(x, x_scale, weight, weight_scale, bias, residual,
                               ACTIVATIONS[activation])


def quantize_rows_fp8(t: Tensor) -> tuple[Tensor, Tensor]:
    """``(values, scales)`` of a matrix ``t`` [..., K]: ``float8_e4m3fn`` rows and their fp32 scales
    max|row| / 448 (a zero row: scale 0, values 0).  What a serving program does once to its
    weights."""
    if t.ndim < 1 or t.shape[-1] < 1:
        raise ValueError(f"t must have shape [..., K], got {tuple(t.shape)}")
    if t.dtype not in DTYPES:
        raise TypeError(f"t must be float32 or bfloat16, got {t.dtype}")
    require_cuda("quantize_rows_fp8", t)
    return native().quantize(t)


__all__ = ["ACTIVATIONS", "linear_act", "linear_act_fp8", "quantize_rows_fp8"]
