"""The torch.library ops' outputs without a gradient (the norm's rstd, the linear's pre-activation) say so:
a loss that uses one must not silently miss its part."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lnet_b200  # noqa: F401

ops = torch.ops.lnet_b200


def outputs(device):
    x = torch.ones(3, 96, dtype=torch.bfloat16, device=device, requires_grad=True)
    w = torch.ones(96, device=device, requires_grad=True)
    up = torch.ones(64, 96, dtype=torch.bfloat16, device=device, requires_grad=True)
    return x, w, up


def check(device):
    x, w, up = outputs(device)
    y, stream, rstd = ops.residual_rms_norm(x, w, x.detach())
    assert y.requires_grad and stream.requires_grad and not rstd.requires_grad
    y, stream, rstd = ops.residual_rms_norm(x, w)
    assert y.requires_grad and not stream.requires_grad and not rstd.requires_grad
    for activation in ("none", "gelu"):
        y, pre = ops.linear_act(x, up, None, None, activation)
        assert y.requires_grad and not pre.requires_grad


def test_fake_outputs():
    with FakeTensorMode():
        check("cpu")


@pytest.mark.gpu
def test_outputs(cuda_device):
    check(cuda_device)
    x, w, up = outputs(cuda_device)
    y, _, rstd = ops.residual_rms_norm(x, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(rstd.sum(), x)
    _, pre = ops.linear_act(x, up, None, None, "gelu")
    with pytest.raises(RuntimeError):
        torch.autograd.grad(pre.sum(), x)
    # the gradients of the others stay what they are
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    y2, _ = lnet_b200.residual_rms_norm(x, w)
    dx2, dw2 = torch.autograd.grad(y2, [x, w], torch.ones_like(y))
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.gpu
def test_opcheck_with_autograd(cuda_device):
    x, w, up = outputs(cuda_device)
    z = torch.randn(4, 100, device=cuda_device, requires_grad=True)
    t, ix = torch.topk(z.detach(), 8)
    for op, args in ((ops.residual_rms_norm, (x, w, x.detach())), (ops.residual_rms_norm, (x, w)),
                     (ops.linear_act, (x, up, None, None, "relu")), (ops.linear_act, (x, up)),
                     (ops.distillation_loss, (z, ix, t))):
        torch.library.opcheck(op.default, args,
                              test_utils=("test_schema", "test_autograd_registration",
                                          "test_faketensor"))
