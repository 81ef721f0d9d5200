"""Refusals of the feed-forward and distillation operators, before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lnet_b200 import (_lib, distillation_loss, residual_rms_norm, residual_rms_norm_fp8)


@pytest.mark.parametrize("norm", [residual_rms_norm, residual_rms_norm_fp8])
def test_norm_refusals(norm):
    x, w = torch.zeros(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA only"):
        norm(x, w)
    with pytest.raises(ValueError, match="weight must have shape"):
        norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="residual must have shape"):
        norm(x, w, torch.zeros(8))
    with pytest.raises(TypeError, match="residual must be"):
        norm(x, w, x.bfloat16())
    with pytest.raises(TypeError, match="x must be"):
        norm(x.half(), w)
    with pytest.raises(TypeError, match="weight must be"):
        norm(x, w.double())
    with pytest.raises(ValueError, match="x must have shape"):
        norm(torch.zeros(()), w)
    with pytest.raises(ValueError, match="eps"):
        norm(x, w, None, -1.0)
    with pytest.raises(ValueError, match="eps"):
        norm(x, w, None, float("nan"))


def test_distillation_refusals():
    z, ix = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64)
    t, lab = torch.zeros(3, 2), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA only"):
        distillation_loss(z, ix, t)
    for bad in (torch.zeros(2, 2, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="teacher_indices"):
            distillation_loss(z, bad, t)
    with pytest.raises(ValueError, match="teacher_logits"):
        distillation_loss(z, ix, torch.zeros(3, 3))
    with pytest.raises(TypeError, match="teacher_indices"):
        distillation_loss(z, ix.int(), t)
    with pytest.raises(TypeError, match="teacher_logits"):
        distillation_loss(z, ix, t.half())
    with pytest.raises(TypeError, match="logits must be"):
        distillation_loss(z.half(), ix, t)
    with pytest.raises(ValueError, match="labels must have shape"):
        distillation_loss(z, ix, t, labels=lab[:2], alpha=0.5)
    with pytest.raises(TypeError, match="labels"):
        distillation_loss(z, ix, t, labels=lab.int(), alpha=0.5)
    with pytest.raises(ValueError, match="pass labels"):
        distillation_loss(z, ix, t, alpha=0.5)
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            distillation_loss(z, ix, t, temperature=tau)
    for alpha in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="alpha"):
            distillation_loss(z, ix, t, labels=lab, alpha=alpha)
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(z, ix, t, reduction="batchmean")


def test_c_entries_refuse_before_any_cuda_call():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    p = ctypes.c_void_p(256)  # never dereferenced: the call is refused first
    assert lib.lnet_b200_residual_rms_norm(p, None, p, _lib.LNET_F64, 0, 4, 8, 0.0, p, None, None,
                                           None) == _lib.LNET_ERR_UNSUPPORTED
    assert lib.lnet_b200_residual_rms_norm(p, p, p, 0, 0, 4, 8, 0.0, p, None, None,
                                           None) == _lib.LNET_ERR_INVALID_ARGUMENT
    assert "stream_out" in _lib.last_error()
    assert lib.lnet_b200_residual_rms_norm_workspace_size(
        0, 1 << 40, 1 << 20, ctypes.byref(n)) == _lib.LNET_ERR_INVALID_ARGUMENT
    assert lib.lnet_b200_residual_rms_norm_workspace_size(
        0, 100, 96, ctypes.byref(n)) == _lib.LNET_OK and n.value >= 96 * 4
    assert lib.lnet_b200_residual_rms_norm_backward(p, p, p, p, None, 0, 0, 100, 96, p, p, None, 0,
                                                    None) == _lib.LNET_ERR_WORKSPACE
    req = _lib.DistillRequest(rows=4, classes=10, top=2, dtype=0, reduction=2, logits=256,
                              teacher_indices=256, teacher_logits=256, labels=None,
                              temperature=1.0, alpha=1.0)
    assert lib.lnet_b200_distill_workspace_size(ctypes.byref(req), ctypes.byref(n)) == _lib.LNET_OK
    assert n.value > 0
    assert lib.lnet_b200_distill_forward(ctypes.byref(req), None, 0, p, None,
                                         None) == _lib.LNET_ERR_WORKSPACE
    for field, value in (("classes", 0), ("temperature", 0.0), ("alpha", 2.0), ("reduction", 3),
                         ("logits", None), ("rows", -1), ("classes", 1 << 31)):
        bad = _lib.DistillRequest.from_buffer_copy(req)
        setattr(bad, field, value)
        assert lib.lnet_b200_distill_workspace_size(
            ctypes.byref(bad), ctypes.byref(n)) == _lib.LNET_ERR_INVALID_ARGUMENT, field
    assert lib.lnet_b200_distill_scale(None, 0, 4, p, None) == _lib.LNET_ERR_INVALID_ARGUMENT
