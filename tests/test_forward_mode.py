"""Forward-mode derivatives and traces: the operators have neither, and say so (a derivative of 0, or a
trace without the launch, would be silent)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from lnet_b200 import _native

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def entries():
    """(entry, arguments, position of each tensor that a derivative may come through)"""
    x, w = torch.zeros(3, 8), torch.ones(8)
    xb, wb, b, r = (torch.zeros(s, dtype=BF) for s in ((3, 8), (5, 8), (5,), (3, 5)))
    xs, ws = torch.ones(3), torch.ones(5)
    z, ix, t = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    return [
        ("norm", (x, w, x.clone(), 1e-6), (0, 1, 2)),
        ("norm_forward", (x, w, x.clone(), 1e-6), (0, 1, 2)),
        ("norm_backward", (x, xs, w, x.clone(), x.clone()), (0, 2, 3, 4)),
        ("norm_fp8", (x, w, x.clone(), 1e-6), (0, 1, 2)),
        ("quantize", (x,), (0,)),
        ("linear", (xb, wb, b, r, 3), (0, 1, 2, 3)),
        ("linear_forward", (xb, wb, b, r, 3), (0, 1, 2, 3)),
        ("linear_backward", (xb, wb, 0, None, r), (0, 1, 4)),
        ("linear_fp8", (xb.to(E4), xs, wb.to(E4), ws, b, r, 0), (1, 3, 4, 5)),
        ("distill", (z, ix, t, None, 1.0, 1.0, 2), (0, 2)),
        ("distill_backward", (z, ix, t, None, 1.0, 1.0, 2, torch.ones(())), (0, 2, 7)),
    ]


CASES = [(name, args, at) for name, args, ats in entries() for at in ats]


@pytest.mark.parametrize("name,args,at", CASES, ids=[f"{n}-{a}" for n, _, a in CASES])
def test_a_forward_gradient_is_refused(name, args, at):
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            getattr(_native.native(), name)(*args[:at], dual, *args[at + 1:])


@pytest.mark.parametrize("name,args", [(n, a) for n, a, _ in entries()],
                         ids=[n for n, _, _ in entries()])
def test_a_trace_is_refused(name, args):
    def call(t):
        out = getattr(_native.native(), name)(t, *args[1:])
        return out if isinstance(out, torch.Tensor) else out[0]

    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, args[0])


@pytest.mark.gpu
def test_public_calls_and_ops(cuda_device):
    import lnet_b200

    ops = torch.ops.lnet_b200
    x = torch.randn(4, 96, device=cuda_device)
    w, xb = torch.ones(96, device=cuda_device), x.to(BF)
    up = torch.randn(64, 96, device=cuda_device).to(BF)
    index = torch.zeros(4, 1, dtype=torch.int64, device=cuda_device)
    teacher = torch.zeros(4, 1, device=cuda_device)
    calls = [(x, lambda t: lnet_b200.residual_rms_norm(t, w)),
             (x, lambda t: lnet_b200.residual_rms_norm_fp8(t, w)),
             (xb, lambda t: lnet_b200.linear_act(t, up)),
             (x, lambda t: lnet_b200.quantize_rows_fp8(t)),
             (x, lambda t: lnet_b200.distillation_loss(t, index, teacher)),
             (x, lambda t: ops.residual_rms_norm(t, w)),
             (x, lambda t: ops.residual_rms_norm_fp8(t, w)),
             (xb, lambda t: ops.linear_act(t, up)),
             (x, lambda t: ops.distillation_loss(t, index, teacher))]
    for i, (t, call) in enumerate(calls):
        for requires_grad in (False, True):
            with forward_ad.dual_level(), torch.set_grad_enabled(requires_grad):
                primal = t.clone().requires_grad_(requires_grad)
                dual = forward_ad.make_dual(primal, torch.ones_like(t))
                try:
                    call(dual)
                except RuntimeError:
                    continue
                pytest.fail(f"call {i}, requires_grad {requires_grad}: a derivative was passed by")
        call(t)  # and without a tangent it runs


@pytest.mark.gpu
def test_a_forward_gradient_through_the_backward_pass_is_refused(cuda_device):
    import lnet_b200

    x = torch.randn(4, 96, device=cuda_device, requires_grad=True)
    w = torch.ones(96, device=cuda_device)
    xb = torch.randn(4, 96, device=cuda_device).to(BF).requires_grad_()
    up = torch.randn(64, 96, device=cuda_device).to(BF)
    index = torch.zeros(4, 1, dtype=torch.int64, device=cuda_device)
    teacher = torch.zeros(4, 1, device=cuda_device)
    for t, out in ((x, lnet_b200.residual_rms_norm(x, w)[0]), (xb, lnet_b200.linear_act(xb, up)),
                   (x, lnet_b200.distillation_loss(x, index, teacher)),
                   (x, lnet_b200.distillation_loss(x, index, teacher, reduction="none"))):
        up_grad = torch.ones_like(out.detach())
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, t, forward_ad.make_dual(up_grad, up_grad))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_the_ops_can_be_traced(cuda_device):
    import lnet_b200

    x = torch.randn(4, 96, device=cuda_device)
    w = torch.ones(96, device=cuda_device)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: lnet_b200.residual_rms_norm(t, w)[0], x)
    traced = torch.jit.trace(lambda t: torch.ops.lnet_b200.residual_rms_norm(t, w)[0], x,
                             check_trace=False)
    other = torch.randn(4, 96, device=cuda_device)
    assert torch.equal(traced(other), lnet_b200.residual_rms_norm(other, w)[0])
