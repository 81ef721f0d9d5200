"""Distillation from a teacher's top logits, with its gradient.

The reference trains its classifiers on hard labels alone
(``torch.nn.functional.cross_entropy`` in its training scripts,
scripts/train_alphabet2d_imagenet100.py); this is the loss for a student of a
teacher whose largest logits were stored: both losses and their gradient in one
pass over the student's logits.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._native import DTYPES, native, require_cuda

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

    A reduced loss takes its gradient in the forward pass, while the logits are on chip, and keeps it
    (as much memory as the logits) for the backward pass, which multiplies it by the loss's own gradient:
    where that is not 1 (a loss scale, a weight), a bfloat16 gradient has been rounded before and after,
    half a unit in the last place each time.  The teacher's logits get no gradient.

    The work grows with V and, for a gradient, with K V / 4096 where K is above 256 (K^2 below).

    Classes masked to -inf have no mass; where the teacher gives one mass, the loss is +inf.  A row
    without an entry or a label has loss and gradient 0, whatever its logits are (NaN, infinities).  An
    index or label past V makes its row's loss and gradient NaN.
    """
    _check_distill_args(logits, teacher_indices, teacher_logits, labels, temperature, alpha,
                        reduction)
    require_cuda("distillation_loss", logits)
    return native().distill(logits, teacher_indices, teacher_logits, labels, temperature, alpha,
                            REDUCTIONS[reduction])


__all__ = ["distillation_loss"]
