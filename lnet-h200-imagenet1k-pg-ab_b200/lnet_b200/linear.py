"""Matrix product with bias, activation and residual in its epilogue.

The reference's channel mixing goes through ``torch.nn.Linear`` (the affine
readout, src/lnet/alphabet.py:49-63); these functions are the layer of a
feed-forward block: ``y = f(x W^T + bias) + residual`` in one kernel on tcgen05,
with its gradient, and its serving form on 8-bit operands
(:func:`lnet_b200.residual_rms_norm_fp8` writes them).
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch import Tensor

from . import _lib
from ._launch import DTYPES, call, pointer, require_cuda, single_backward, wants_grad

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


def _request(x, weight, bias, residual, activation, x_scale=None,
             weight_scale=None) -> _lib.LinearRequest:
    return _lib.LinearRequest(
        x.numel() // x.shape[-1], x.shape[-1], weight.shape[0],
        _lib.LNET_BF16 if x.dtype == torch.bfloat16 else _lib.LNET_E4M3, activation,
        x.data_ptr(), weight.data_ptr(), pointer(bias), pointer(residual), pointer(x_scale),
        pointer(weight_scale))


# Workspace sizes depend on the extents, the type and the alignment of the pointers alone.
@lru_cache(maxsize=1024)
def _forward_bytes(rows, inner, outer, dtype, x_align, w_align) -> int:
    n = ctypes.c_size_t(0)
    req = _lib.LinearRequest(rows, inner, outer, dtype, 0, 256 + x_align, 256 + w_align, None,
                             None, 256, 256)
    _lib.check(_lib.load().lnet_b200_linear_workspace_size(ctypes.byref(req), ctypes.byref(n)),
               "lnet_b200_linear_workspace_size")
    return int(n.value)


@lru_cache(maxsize=1024)
def _backward_bytes(rows, inner, outer, activation, x_align, w_align, pre_align, dy_align,
                    want_dx, want_dw, want_db) -> int:
    n = ctypes.c_size_t(0)
    req = _lib.LinearRequest(rows, inner, outer, _lib.LNET_BF16, activation, 256 + x_align,
                             256 + w_align)
    _lib.check(_lib.load().lnet_b200_linear_backward_workspace_size(
        ctypes.byref(req), 256 + pre_align if activation else None, 256 + dy_align, want_dx,
        want_dw, want_db, ctypes.byref(n)), "lnet_b200_linear_backward_workspace_size")
    return int(n.value)


def _workspace(nbytes: int, device: torch.device) -> Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _launch_linear(x, req, keep_preact: bool) -> tuple[Tensor, Tensor | None]:
    """(y, pre-activation or None) of a request of contiguous tensors."""
    device = x.device
    nbytes = _forward_bytes(req.rows, req.inner, req.outer, req.dtype, (req.x or 0) & 15,
                            req.weight & 15)
    y = torch.empty((*x.shape[:-1], req.outer), dtype=torch.bfloat16, device=device)
    pre = torch.empty_like(y) if keep_preact else None
    ws = _workspace(nbytes, device)
    call(device, "lnet_b200_linear_forward", ctypes.byref(req), pointer(ws), nbytes, y.data_ptr(),
         pointer(pre))
    return y, pre


def _launch_linear_backward(x, weight, activation, pre, dy, want_dx, want_dw, want_db):
    """(dx, dweight, dbias), each None where it is not wanted."""
    req = _request(x, weight, None, None, activation)
    pre_at, dy_at = pointer(pre), dy.data_ptr()
    nbytes = _backward_bytes(req.rows, req.inner, req.outer, activation, (req.x or 0) & 15,
                             req.weight & 15, (pre_at or 0) & 15, dy_at & 15, want_dx, want_dw,
                             want_db)
    dx = torch.empty_like(x) if want_dx else None
    dw = torch.empty_like(weight) if want_dw else None
    db = torch.empty(req.outer, dtype=torch.bfloat16, device=x.device) if want_db else None
    ws = _workspace(nbytes, x.device)
    call(x.device, "lnet_b200_linear_backward", ctypes.byref(req), pre_at, dy_at, pointer(ws),
         nbytes, pointer(dx), pointer(dw), pointer(db))
    return dx, dw, db


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        xc, wc = x.contiguous(), weight.contiguous()
        bc = None if bias is None else bias.contiguous()
        rc = None if residual is None else residual.contiguous()
        code = ACTIVATIONS[activation]
        needs = ctx.needs_input_grad
        slope = code != 0 and (needs[0] or needs[1] or needs[2])
        y, pre = _launch_linear(xc, _request(xc, wc, bc, rc, code), slope)
        ctx.save_for_backward(xc, wc, pre)
        ctx.activation = code
        return y

    @staticmethod
    @single_backward
    def backward(ctx, dy):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            dx, dw, db = _launch_linear_backward(x, weight, ctx.activation, pre, dy.contiguous(),
                                                 need_x, need_w, need_b)
        return dx, dw, db, dy if need_r else None, None


def linear_act(x: Tensor, weight: Tensor, bias: Tensor | None = None,
               residual: Tensor | None = None, *, activation: str = "none") -> Tensor:
    """``f(x @ weight.T + bias) + residual`` for bfloat16 ``x`` [..., K] and ``weight`` [N, K].

    ``activation`` is ``"none"``, ``"relu"``, ``"silu"`` or ``"gelu"`` (the erf form).  Sums are
    fp32 and the result is rounded once to bfloat16.  Differentiable in ``x``, ``weight``, ``bias``
    and ``residual``; through an activation the forward pass keeps x W^T + bias in bfloat16.
    """
    _check_linear_args(x, weight, bias, residual, activation, torch.bfloat16)
    require_cuda("linear_act", x)
    if wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, activation)
    x, weight = x.contiguous(), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    return _launch_linear(x, _request(x, weight, bias, residual, ACTIVATIONS[activation]),
                          False)[0]


def linear_act_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor,
                   bias: Tensor | None = None, residual: Tensor | None = None, *,
                   activation: str = "none") -> Tensor:
    """:func:`linear_act` on 8-bit operands: ``x`` [..., K] and ``weight`` [N, K] are
    ``float8_e4m3fn`` with the fp32 scales ``x_scale`` [...] and ``weight_scale`` [N] of their rows
    (:func:`lnet_b200.residual_rms_norm_fp8`, :func:`quantize_rows_fp8`); bias, residual and the
    result are bfloat16.  A serving form: it has no gradient and refuses inputs that want one.
    """
    _check_linear_args(x, weight, bias, residual, activation, torch.float8_e4m3fn)
    for name, t, shape in (("x_scale", x_scale, tuple(x.shape[:-1])),
                           ("weight_scale", weight_scale, (weight.shape[0],))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    require_cuda("linear_act_fp8", x)
    if wants_grad(x, x_scale, weight, weight_scale, bias, residual):
        raise RuntimeError("linear_act_fp8 has no gradient: call it under torch.no_grad()")
    x, weight = x.contiguous(), weight.contiguous()
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    return _launch_linear(x, _request(x, weight, bias, residual, ACTIVATIONS[activation], x_scale,
                                      weight_scale), False)[0]


def quantize_rows_fp8(t: Tensor) -> tuple[Tensor, Tensor]:
    """``(values, scales)`` of a matrix ``t`` [..., K]: ``float8_e4m3fn`` rows and their fp32 scales
    max|row| / 448 (a zero row: scale 0, values 0).  What a serving program does once to its
    weights."""
    if t.ndim < 1 or t.shape[-1] < 1:
        raise ValueError(f"t must have shape [..., K], got {tuple(t.shape)}")
    if t.dtype not in DTYPES:
        raise TypeError(f"t must be float32 or bfloat16, got {t.dtype}")
    require_cuda("quantize_rows_fp8", t)
    t = t.detach().contiguous()
    values = torch.empty(t.shape, dtype=torch.float8_e4m3fn, device=t.device)
    scales = torch.empty(t.shape[:-1], dtype=torch.float32, device=t.device)
    call(t.device, "lnet_b200_quantize_rows_fp8", t.data_ptr(), DTYPES[t.dtype],
         t.numel() // t.shape[-1], t.shape[-1], values.data_ptr(), scales.data_ptr())
    return values, scales


__all__ = ["ACTIVATIONS", "linear_act", "linear_act_fp8", "quantize_rows_fp8"]
