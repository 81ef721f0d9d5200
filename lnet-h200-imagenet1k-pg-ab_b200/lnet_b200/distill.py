"""Distillation from a teacher's top logits, with its gradient.

The reference trains its classifiers on hard labels alone
(``torch.nn.functional.cross_entropy`` in its training scripts,
scripts/train_alphabet2d_imagenet100.py); this is the loss for a student of a
teacher whose largest logits were stored: both losses and their gradient in one
pass over the student's logits.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch import Tensor

from . import _lib
from ._launch import DTYPES, call, pointer, require_cuda, single_backward, wants_grad

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _check_distill_args(logits, teacher_indices, teacher_logits, labels, temperature, alpha,
                        reduction) -> None:
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., V], got {tuple(logits.shape)}")
    if logits.dtype not in DTYPES:
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    lead = tuple(logits.shape[:-1])
    if teacher_indices.ndim != logits.ndim or tuple(teacher_indices.shape[:-1]) != lead:
        raise ValueError(f"teacher_indices must have shape {(*lead, 'K')}, "
                         f"got {tuple(teacher_indices.shape)}")
    if teacher_logits.shape != teacher_indices.shape:
        raise ValueError(f"teacher_logits must have shape {tuple(teacher_indices.shape)}, "
                         f"got {tuple(teacher_logits.shape)}")
    if teacher_indices.dtype != torch.int64:
        raise TypeError(f"teacher_indices must be int64, got {teacher_indices.dtype}")
    if teacher_logits.dtype not in DTYPES:
        raise TypeError(f"teacher_logits must be float32 or bfloat16, got {teacher_logits.dtype}")
    if labels is None:
        if alpha != 1.0:
            raise ValueError(f"alpha {alpha} mixes labels in: pass labels, or alpha 1")
    else:
        if tuple(labels.shape) != lead:
            raise ValueError(f"labels must have shape {lead}, got {tuple(labels.shape)}")
        if labels.dtype != torch.int64:
            raise TypeError(f"labels must be int64, got {labels.dtype}")
    for name, t in (("teacher_indices", teacher_indices), ("teacher_logits", teacher_logits),
                    ("labels", labels)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, logits on {logits.device}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"alpha must lie in [0, 1], got {alpha}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(REDUCTIONS)}, got {reduction!r}")


@lru_cache(maxsize=256)
def _workspace_bytes(rows: int, top: int, reduction: int) -> int:
    n = ctypes.c_size_t(0)
    req = _lib.DistillRequest(rows=rows, classes=1, top=top, reduction=reduction, logits=1,
                              teacher_indices=1, teacher_logits=1, temperature=1.0,
                              alpha=1.0)  # the size depends on nothing else
    _lib.check(_lib.load().lnet_b200_distill_workspace_size(ctypes.byref(req), ctypes.byref(n)),
               "lnet_b200_distill_workspace_size")
    return int(n.value)


class _Request:
    """One call's request and workspace (the tensors are kept for its pointers)."""

    def __init__(self, logits, indices, teacher, labels, temperature, alpha, reduction):
        self.keep = (logits, indices, teacher, labels)
        self.device = logits.device
        self.req = _lib.DistillRequest(
            rows=logits.numel() // logits.shape[-1], classes=logits.shape[-1],
            top=indices.shape[-1], dtype=DTYPES[logits.dtype], reduction=reduction,
            logits=logits.data_ptr(), teacher_indices=indices.data_ptr(),
            teacher_logits=teacher.data_ptr(), labels=pointer(labels), temperature=temperature,
            alpha=alpha)

    def run(self, name, *args):
        nbytes = _workspace_bytes(self.req.rows, self.req.top, self.req.reduction)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        call(self.device, name, ctypes.byref(self.req), ws.data_ptr(), nbytes, *args)


def _launch_distill(logits, indices, teacher, labels, temperature, alpha, reduction,
                    want_grad) -> tuple[Tensor, Tensor | None]:
    """(loss, gradient of the reduced loss or None) of contiguous tensors."""
    shape = logits.shape[:-1] if reduction == 0 else ()
    loss = torch.empty(shape, dtype=torch.float32, device=logits.device)
    dlogits = torch.empty_like(logits) if want_grad else None
    _Request(logits, indices, teacher, labels, temperature, alpha, reduction).run(
        "lnet_b200_distill_forward", loss.data_ptr(), pointer(dlogits))
    return loss, dlogits


class _DistillationLoss(torch.autograd.Function):
    """A reduced loss takes its gradient in the forward pass, while the logits are on chip
    or in L2; the backward pass scales it in place by the loss's gradient (a launch that reads
    one value where that is 1).  The rows' losses (``none``), and a second backward pass, take
    the gradient from the logits again."""

    @staticmethod
    def forward(ctx, logits, indices, teacher, labels, temperature, alpha, reduction):
        args = (logits.contiguous(), indices.contiguous(), teacher.float().contiguous(),
                None if labels is None else labels.contiguous())
        loss, dlogits = _launch_distill(*args, temperature, alpha, reduction, reduction != 0)
        ctx.save_for_backward(*args)
        ctx.scalars = (temperature, alpha, reduction)
        ctx.ready = dlogits
        return loss

    @staticmethod
    @single_backward
    def backward(ctx, dloss):
        args = ctx.saved_tensors
        logits = args[0]
        dloss = dloss.float().contiguous()
        dlogits, ctx.ready = ctx.ready, None
        if dlogits is not None:
            call(logits.device, "lnet_b200_distill_scale", dlogits.data_ptr(),
                 DTYPES[logits.dtype], dlogits.numel(), dloss.data_ptr())
        else:
            dlogits = torch.empty_like(logits)
            _Request(*args, *ctx.scalars).run("lnet_b200_distill_backward", dloss.data_ptr(),
                                              dlogits.data_ptr())
        return dlogits, None, None, None, None, None, None


def distillation_loss(logits: Tensor, teacher_indices: Tensor, teacher_logits: Tensor, *,
                      labels: Tensor | None = None, temperature: float = 1.0, alpha: float = 1.0,
                      reduction: str = "mean") -> Tensor:
    """Loss of a student's ``logits`` [..., V] (float32 or bfloat16) against a teacher's top
    entries: ``alpha * temperature^2 * KL(p || q) + (1 - alpha) * cross entropy(labels)``.

    ``p`` is the softmax of ``teacher_logits`` [..., K] at ``temperature`` over the kept entries
    and ``q`` the student's softmax at ``temperature`` over all V classes; an entry with a negative
    index in ``teacher_indices`` [..., K] (int64), or with a logit of -inf, is padding.  ``labels``
    [...] (int64) may hold negative values for rows without one.  ``reduction`` is ``"none"``
    (the rows' losses), ``"sum"`` or ``"mean"`` (over the rows that have an entry or a label; 0
    where none has).  The loss is fp32; it is differentiable in ``logits``.

    Classes masked to -inf have no mass; where the teacher gives one mass, the loss is +inf.  An
    index or label past V makes its row's loss and gradient NaN.
    """
    _check_distill_args(logits, teacher_indices, teacher_logits, labels, temperature, alpha,
                        reduction)
    require_cuda("distillation_loss", logits)
    code = REDUCTIONS[reduction]
    if wants_grad(logits):
        return _DistillationLoss.apply(logits, teacher_indices, teacher_logits, labels,
                                       float(temperature), float(alpha), code)
    loss, _ = _launch_distill(logits.contiguous(), teacher_indices.contiguous(),
                              teacher_logits.float().contiguous(),
                              None if labels is None else labels.contiguous(),
                              float(temperature), float(alpha), code, False)
    return loss


__all__ = ["distillation_loss"]
