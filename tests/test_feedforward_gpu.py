"""The feed-forward block, its 8-bit form, the torch.library ops and the example that runs them together."""

from __future__ import annotations

import importlib.util
import math

import pytest
import torch
from conftest import ROOT

import lnet_b200
from lnet_b200 import B200FeedForward

pytestmark = pytest.mark.gpu

ops = torch.ops.lnet_b200


def make(shape, seed, device, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).bfloat16().to(device)


def reference(block, x, residual):
    """The block in 64 bits from its own parameters."""
    h = x.double() if residual is None else (x.float() + residual.float()).bfloat16().double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + block.eps) * block.norm_weight.double()
    a = y @ block.up.weight.double().t() + block.up.bias.double()
    u = 0.5 * a * (1 + torch.erf(a / math.sqrt(2)))
    return u @ block.down.weight.double().t() + block.down.bias.double() + h


@pytest.mark.parametrize("shape", [(1, 96), (7, 96), (3, 50, 96), (2, 1000, 96)])
def test_block(shape, cuda_device):
    torch.manual_seed(0)
    block = B200FeedForward(96, 384, device=cuda_device)
    x, r = make(shape, 1, cuda_device), make(shape, 2, cuda_device)
    ref = reference(block, x, r).detach()
    out = block(x, r).detach()
    # three roundings to bf16 of half a unit, 2^-8, on values whose sums of 384 products are no
    # larger than the result's own scale
    assert float((out.double() - ref).abs().max()) <= 3 * 2.0 ** -8 * float(ref.abs().max())
    served = block.quantize_()(x, r)
    # e4m3 rows: 2^-4 an element at most, in random directions over the sums: well below 2^-4 of
    # the branch
    branch = (ref - (x.float() + r.float()).bfloat16().double()).norm()
    assert float((served.double() - ref).norm()) <= 2.0 ** -4 * float(branch) + \
        2.0 ** -8 * float(ref.norm())
    block.train()
    assert torch.equal(block(x, r), out)


def test_block_trains(cuda_device):
    torch.manual_seed(0)
    block = B200FeedForward(96, 384, device=cuda_device)
    x = make((40, 96), 1, cuda_device).requires_grad_()
    r = make((40, 96), 2, cuda_device).requires_grad_()
    dy = make((40, 96), 3, cuda_device)
    params = list(block.parameters())
    grads = torch.autograd.grad(block(x, r), [x, r, *params], dy)
    want = torch.autograd.grad(reference(block, x, r), [x, r, *params], dy.double())
    for g, ref in zip(grads, want):
        # roundings of the activations, of da and of the result: a few 2^-8 of the gradient's norm
        assert float((g.double() - ref.double()).norm()) <= 4 * 2.0 ** -8 * float(ref.norm())


def test_ops_match_the_functions(cuda_device):
    x, r = make((33, 96), 1, cuda_device), make((33, 96), 2, cuda_device)
    w = torch.rand(96, device=cuda_device) + 0.5
    y, h = lnet_b200.residual_rms_norm(x, w, r)
    y2, h2, _ = ops.residual_rms_norm(x, w, r)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    up, b = make((384, 96), 3, cuda_device, 0.1), make((384,), 4, cuda_device)
    u = lnet_b200.linear_act(y, up, b, activation="gelu")
    assert torch.equal(u, ops.linear_act(y, up, b, None, "gelu")[0])
    q, s, _ = lnet_b200.residual_rms_norm_fp8(x, w, r)
    q2, s2, _ = ops.residual_rms_norm_fp8(x, w, r)
    assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)
    uq, us = lnet_b200.quantize_rows_fp8(up)
    assert torch.equal(lnet_b200.linear_act_fp8(q, s, uq, us, b),
                       ops.linear_act_fp8(q, s, uq, us, b))
    z = torch.randn(12, 1000, device=cuda_device)
    t, ix = torch.topk(z + 1, 8)
    assert torch.equal(lnet_b200.distillation_loss(z, ix, t, temperature=2.0),
                       ops.distillation_loss(z, ix, t, None, 2.0))


def test_op_gradients_match_the_functions(cuda_device):
    x = make((33, 96), 1, cuda_device).requires_grad_()
    r = make((33, 96), 2, cuda_device).requires_grad_()
    w = (torch.rand(96, device=cuda_device) + 0.5).requires_grad_()
    dy, dh = make((33, 96), 5, cuda_device), make((33, 96), 6, cuda_device)
    one = torch.autograd.grad(lnet_b200.residual_rms_norm(x, w, r), [x, r, w], [dy, dh])
    two = torch.autograd.grad(ops.residual_rms_norm(x, w, r)[:2], [x, r, w], [dy, dh])
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    up = make((64, 96), 3, cuda_device, 0.1).requires_grad_()
    b = make((64,), 4, cuda_device).requires_grad_()
    du = make((33, 64), 7, cuda_device)
    one = torch.autograd.grad(lnet_b200.linear_act(x, up, b, activation="silu"), [x, up, b], du)
    two = torch.autograd.grad(ops.linear_act(x, up, b, None, "silu")[0], [x, up, b], du)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    z = torch.randn(12, 1000, device=cuda_device, requires_grad=True)
    t, ix = torch.topk(z.detach() + 1, 8)
    one, = torch.autograd.grad(lnet_b200.distillation_loss(z, ix, t, temperature=2.0), z)
    two, = torch.autograd.grad(ops.distillation_loss(z, ix, t, None, 2.0), z)
    assert torch.equal(one, two)


def test_opcheck(cuda_device):
    x = make((5, 96), 1, cuda_device)
    w = torch.ones(96, device=cuda_device)
    up = make((64, 96), 3, cuda_device)
    z = torch.randn(4, 100, device=cuda_device)
    t, ix = torch.topk(z, 8)
    for op, args in ((ops.residual_rms_norm, (x, w, x.clone())), (ops.residual_rms_norm, (x, w)),
                     (ops.linear_act, (x, up, None, None, "relu")), (ops.linear_act, (x, up)),
                     (ops.distillation_loss, (z, ix, t))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


def test_example(cuda_device):
    spec = importlib.util.spec_from_file_location("distill_feedforward",
                                                  ROOT / "examples" / "distill_feedforward.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    out = m.run(steps=25, batch=32, log=lambda *_: None)
    assert out["losses"][-1] < 0.5 * out["losses"][0]
    assert out["fp8"] < 0.2 and out["single"] < 0.05
