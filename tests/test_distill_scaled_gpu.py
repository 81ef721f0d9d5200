"""A reduced distillation loss whose own gradient is not 1, and strided arguments; tolerances of
test_distill_gpu."""

from __future__ import annotations

import math

import pytest
import torch
from test_distill_gpu import DTYPES, FP32, HALF_ULP, make, reference

from lnet_b200 import distillation_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes", [(8, 1000), (7, 1001), (3, 40003)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("factor", [0.25, 3.0, 0.3])
def test_the_first_backward_of_a_scaled_loss(factor, reduction, rows, classes, dtype, cuda_device):
    """The gradient taken with the loss, times the loss's own gradient: in bf16 rounded before and after."""
    z, index, teacher, labels = make(rows, classes, 9, dtype, 3, cuda_device)
    tau, alpha = 2.0, 0.5
    zg = z.clone().requires_grad_()
    loss = distillation_loss(zg, index, teacher, labels=labels, temperature=tau, alpha=alpha,
                             reduction=reduction)
    dz, = torch.autograd.grad(factor * loss, zg)
    z64 = z.double().requires_grad_()
    ref, = torch.autograd.grad(reference(z64, index, teacher, labels, tau, alpha, reduction), z64)
    ref = ref * factor
    err = (dz.double() - ref).abs()
    unit = alpha * tau + 1
    if reduction == "mean":
        unit /= int((((index >= 0) & (teacher > -math.inf)).any(-1) | (labels >= 0)).sum())
    tol = 2.01 * HALF_ULP[dtype] * 1.01 * ref.abs() + FP32 * factor * unit
    assert bool((err <= tol).all()), float((err - tol).max())


def test_strided_arguments_give_the_same_values(cuda_device):
    z, index, teacher, labels = make(12, 777, 5, torch.bfloat16, 3, cuda_device)
    kw = dict(temperature=2.0, alpha=0.5)
    wide = torch.full((12, 1000), math.nan, dtype=z.dtype, device=cuda_device)
    wide[:, 3:780] = z
    views = (wide[:, 3:780], index.t().contiguous().t(), teacher.t().contiguous().t())
    lab2 = torch.stack([labels, labels], 1)[:, 0]
    for reduction in ("none", "mean"):
        want = distillation_loss(z, index, teacher, labels=labels, reduction=reduction, **kw)
        got = distillation_loss(*views, labels=lab2, reduction=reduction, **kw)
        assert torch.equal(got, want)
    zg, wg = z.clone().requires_grad_(), wide.clone().requires_grad_()
    dz, = torch.autograd.grad(distillation_loss(zg, index, teacher, labels=labels, **kw), zg)
    dw, = torch.autograd.grad(distillation_loss(wg[:, 3:780], *views[1:], labels=lab2, **kw), wg)
    assert torch.equal(dw[:, 3:780], dz) and bool((dw[:, :3] == 0).all())
