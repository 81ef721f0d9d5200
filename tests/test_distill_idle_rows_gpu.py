"""Rows without a target: loss and gradient 0 whatever their logits are, and the other rows as without them."""

from __future__ import annotations

import math

import pytest
import torch
from test_distill_gpu import DTYPES, make

from lnet_b200 import distillation_loss

pytestmark = pytest.mark.gpu


# a block, an odd row, several blocks, a row that is read twice, more entries than are kept on chip
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes,top", [(5, 2), (1000, 8), (1001, 8), (40001, 8), (100003, 8),
                                         (3001, 400)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tau,alpha", [(2.0, 0.6), (1.0, 1.0), (2.0, 0.0)])
def test_rows_without_a_target(tau, alpha, reduction, classes, top, dtype, cuda_device):
    z, index, teacher, labels = make(8, classes, top, dtype, classes, cuda_device)
    idle = torch.tensor([1, 2, 4, 5, 6], device=cuda_device)
    index[idle], labels[idle], labels[3] = -1, -100, 0
    if classes > 5:
        teacher[6], index[6] = -math.inf, 3  # entries without mass
    kw = dict(labels=labels, temperature=tau, alpha=alpha, reduction=reduction)

    def run(values):
        t = values.clone().requires_grad_()
        loss = distillation_loss(t, index, teacher, **kw)
        return loss.detach(), torch.autograd.grad(loss, t, torch.ones_like(loss))[0]

    want, want_dz = run(z)
    assert bool((want_dz[idle] == 0).all())
    z[1], z[4], z[5] = math.nan, math.inf, -math.inf
    z[2, classes // 2] = math.inf
    z[6, 0] = math.nan
    loss, dz = run(z)
    assert torch.equal(loss, want) and torch.equal(dz, want_dz)
    with torch.no_grad():
        alone = distillation_loss(z, index, teacher, **kw)
    assert bool(torch.isfinite(alone).all())
