"""Tensors without memory of their own (functional wrappers, function transforms): refused, and an optional
argument among them is not taken for a missing one."""

from __future__ import annotations

import pytest
import torch

from lnet_b200 import (distillation_loss, linear_act, linear_act_fp8, quantize_rows_fp8, residual_rms_norm,
                       residual_rms_norm_fp8)

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def calls(device):
    """(a call of one tensor, the tensor), the others being ordinary."""
    x, w = torch.randn(3, 8, device=device), torch.ones(8, device=device)
    r = torch.randn(3, 8, device=device)
    xb, wb, b, rb = (torch.randn(s, device=device).to(BF) for s in ((3, 8), (5, 8), (5,), (3, 5)))
    (xq, xs), (wq, ws) = quantize_rows_fp8(xb), quantize_rows_fp8(wb)
    z, t = torch.randn(3, 8, device=device), torch.randn(3, 2, device=device)
    ix, lab = torch.zeros(3, 2, dtype=torch.int64, device=device), torch.ones(3, dtype=torch.int64,
                                                                             device=device)
    kw = dict(alpha=0.5, temperature=2.0)
    return {
        "norm x": (lambda a: residual_rms_norm(a, w, r)[0], x),
        "norm residual": (lambda a: residual_rms_norm(x, w, a)[0], r),
        "norm fp8 residual": (lambda a: residual_rms_norm_fp8(x, w, a)[1], r),
        "linear x": (lambda a: linear_act(a, wb, b, rb), xb),
        "linear bias": (lambda a: linear_act(xb, wb, a, rb), b),
        "linear residual": (lambda a: linear_act(xb, wb, b, a), rb),
        "linear fp8 bias": (lambda a: linear_act_fp8(xq, xs, wq, ws, a, rb), b),
        "linear fp8 residual": (lambda a: linear_act_fp8(xq, xs, wq, ws, b, a), rb),
        "distillation logits": (lambda a: distillation_loss(a, ix, t, labels=lab, **kw), z),
        "distillation labels": (lambda a: distillation_loss(z, ix, t, labels=a, **kw), lab),
    }


NAMES = ["norm x", "norm residual", "norm fp8 residual", "linear x", "linear bias", "linear residual",
         "linear fp8 bias", "linear fp8 residual", "distillation logits", "distillation labels"]


@pytest.mark.parametrize("name", NAMES)
def test_functional_wrappers(name, cuda_device):
    call, t = calls(cuda_device)[name]
    call(t)
    with pytest.raises(RuntimeError):
        torch.func.functionalize(call)(t)


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms(name, cuda_device):
    call, t = calls(cuda_device)[name]
    with pytest.raises(RuntimeError):
        torch.vmap(call)(torch.stack([t, t]))
    if t.is_floating_point():
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda a: call(a).float().sum())(t)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
