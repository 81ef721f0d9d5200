"""Refusals of the feed-forward and distillation operators, before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from torch._subclasses.fake_tensor import FakeTensorMode

from lnet_b200 import (B200FeedForward, _lib, distillation_loss, linear_act, linear_act_fp8, quantize_rows_fp8,
                       residual_rms_norm, residual_rms_norm_fp8)


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


def test_linear_refusals():
    bf = torch.bfloat16
    x, w, b = torch.zeros(3, 8, dtype=bf), torch.zeros(5, 8, dtype=bf), torch.zeros(5, dtype=bf)
    r = torch.zeros(3, 5, dtype=bf)
    with pytest.raises(RuntimeError, match="CUDA only"):
        linear_act(x, w, b, r)
    with pytest.raises(TypeError, match="x must be"):
        linear_act(x.float(), w)
    with pytest.raises(TypeError, match="weight must be"):
        linear_act(x, w.float())
    for bad in (w[:, :7], w[0], w[:0]):
        with pytest.raises(ValueError, match="weight must have shape"):
            linear_act(x, bad)
    with pytest.raises(ValueError, match="bias must have shape"):
        linear_act(x, w, b[:4])
    with pytest.raises(TypeError, match="bias must be"):
        linear_act(x, w, b.float())
    with pytest.raises(ValueError, match="residual must have shape"):
        linear_act(x, w, b, r[:2])
    with pytest.raises(TypeError, match="residual must be"):
        linear_act(x, w, b, r.float())
    with pytest.raises(ValueError, match="activation"):
        linear_act(x, w, b, activation="tanh")
    e4 = torch.float8_e4m3fn
    xs, ws = torch.ones(3), torch.ones(5)
    with pytest.raises(TypeError, match="x must be"):
        linear_act_fp8(x, xs, w.to(e4), ws)
    with pytest.raises(ValueError, match="x_scale must have shape"):
        linear_act_fp8(x.to(e4), ws, w.to(e4), ws)
    with pytest.raises(TypeError, match="weight_scale must be"):
        linear_act_fp8(x.to(e4), xs, w.to(e4), ws.double())
    with pytest.raises(RuntimeError, match="CUDA only"):
        linear_act_fp8(x.to(e4), xs, w.to(e4), ws)
    with pytest.raises(TypeError, match="t must be"):
        quantize_rows_fp8(torch.zeros(2, 2, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="CUDA only"):
        quantize_rows_fp8(x)


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
    lin = _lib.LinearRequest(rows=100, inner=90, outer=64, dtype=_lib.LNET_BF16, activation=1,
                             x=256, weight=256)
    assert lib.lnet_b200_linear_workspace_size(ctypes.byref(lin), ctypes.byref(n)) == _lib.LNET_OK
    assert n.value >= 164 * 96 * 2  # rows of 180 bytes are copied to rows of 192
    assert lib.lnet_b200_linear_forward(ctypes.byref(lin), None, 0, p, None,
                                        None) == _lib.LNET_ERR_WORKSPACE
    assert lib.lnet_b200_linear_backward(ctypes.byref(lin), None, p, None, 0, p, p, p,
                                         None) == _lib.LNET_ERR_INVALID_ARGUMENT
    assert "preact" in _lib.last_error()
    for field, value, status in (("dtype", _lib.LNET_F32, _lib.LNET_ERR_UNSUPPORTED),
                                 ("dtype", _lib.LNET_E4M3, _lib.LNET_ERR_INVALID_ARGUMENT),
                                 ("activation", 4, _lib.LNET_ERR_INVALID_ARGUMENT),
                                 ("inner", 0, _lib.LNET_ERR_INVALID_ARGUMENT),
                                 ("outer", 1 << 40, _lib.LNET_ERR_INVALID_ARGUMENT),
                                 ("weight", None, _lib.LNET_ERR_INVALID_ARGUMENT)):
        bad = _lib.LinearRequest.from_buffer_copy(lin)
        setattr(bad, field, value)
        assert lib.lnet_b200_linear_workspace_size(ctypes.byref(bad),
                                                   ctypes.byref(n)) == status, field
    assert lib.lnet_b200_distill_scale(None, 0, 4, p, None) == _lib.LNET_ERR_INVALID_ARGUMENT


def test_ops_are_registered_and_functional():
    for name in ("residual_rms_norm", "residual_rms_norm_fp8", "linear_act", "linear_act_fp8",
                 "distillation_loss"):
        schema = str(getattr(torch.ops.lnet_b200, name).default._schema)
        assert "!" not in schema.split("->")[0], schema


def test_fake_shapes_and_errors():
    bf, e4 = torch.bfloat16, torch.float8_e4m3fn
    ops = torch.ops.lnet_b200
    with FakeTensorMode():
        x, w = torch.empty(2, 5, 96, dtype=bf), torch.empty(96)
        y, h, rstd = ops.residual_rms_norm(x, w, x)
        assert y.shape == h.shape == x.shape and y.dtype == bf
        assert rstd.shape == (2, 5) and rstd.dtype == torch.float32
        assert ops.residual_rms_norm(x, w)[1].shape == (0,)
        q, s, h = ops.residual_rms_norm_fp8(x, w, x)
        assert q.dtype == e4 and s.shape == (2, 5) and h.shape == x.shape
        up = torch.empty(384, 96, dtype=bf)
        y, pre = ops.linear_act(x, up, activation="gelu")
        assert y.shape == pre.shape == (2, 5, 384) and y.dtype == bf
        assert ops.linear_act(x, up)[1].shape == (0,)
        y = ops.linear_act_fp8(q, s, torch.empty(384, 96, dtype=e4), torch.empty(384))
        assert y.shape == (2, 5, 384) and y.dtype == bf
        z, ix = torch.empty(2, 5, 1000), torch.empty(2, 5, 8, dtype=torch.int64)
        t = torch.empty(2, 5, 8)
        assert ops.distillation_loss(z, ix, t).shape == ()
        assert ops.distillation_loss(z, ix, t, None, 1.0, 1.0, "none").shape == (2, 5)
        with pytest.raises(ValueError):
            ops.residual_rms_norm(x, torch.empty(95))
        with pytest.raises(TypeError):
            ops.linear_act(x.float(), up)
        with pytest.raises(ValueError):
            ops.distillation_loss(z, ix, t[..., :7])


def test_feedforward_module_on_cpu():
    block = B200FeedForward(96, 384)
    assert {n: tuple(p.shape) for n, p in block.named_parameters()} == {
        "norm_weight": (96,), "up.weight": (384, 96), "up.bias": (384,),
        "down.weight": (96, 384), "down.bias": (96,)}
    with pytest.raises(RuntimeError, match="CUDA only"):
        block(torch.zeros(2, 96, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        B200FeedForward(96, 0)
    with pytest.raises(ValueError):
        B200FeedForward(96, 384, activation="tanh")


def test_request_layouts_match_the_header():
    import re

    from conftest import ROOT

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "lnet_b200.h").read_text(), flags=re.S)
    for name, py in (("lnet_b200_linear_request", _lib.LinearRequest),
                     ("lnet_b200_distill_request", _lib.DistillRequest)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S)
        assert re.findall(r"(\w+)\s*;", body.group(1)) == [f for f, _ in py._fields_]
