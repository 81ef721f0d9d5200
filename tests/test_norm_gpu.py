"""Residual addition + RMSNorm, its gradient and its 8-bit output, against the formula in 64 bits.

Tolerances.  Inputs are exact in the reference, so what is left is fp32 arithmetic and the last
rounding.  A sum of D squares or products over 16 to 32 terms a thread and a tree has a relative
error below (32 + 10) 2^-24 = 2.5e-6 of the sum of magnitudes; FP32 = 4e-6 covers it with the few
products after it.  A bf16 output adds half a unit in the last place, 2^-8 of the value (8 significant bits), and an
e4m3 code half a step, 2^-4 of the value or 2^-10 of the scale below the normals.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import lnet_b200
from lnet_b200 import _lib, residual_rms_norm, residual_rms_norm_fp8

pytestmark = pytest.mark.gpu

FP32 = 4e-6
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}
DTYPES = [torch.float32, torch.bfloat16]
# one element, a lane group of each size, odd widths, a block a row, rows that no block holds, and
# many rows of odd and even widths
SHAPES = [(1, 1), (1, 96), (7, 64), (300, 96), (5, 3, 128), (33, 257), (19, 1001), (64, 1024),
          (9, 4096), (3, 8200), (2, 8193), (2, 16392), (2, 20001), (1300, 2048), (1201, 4096),
          (1211, 1544), (3001, 97), (2500, 1001), (700, 2049), (20011, 33),
          (300, 6795), (2100, 5001), (40, 12003)]


def make(shape, dtype, seed, device, std=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


def stream_of(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def norm64(h, w, eps):
    h64 = h.double()
    return h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + eps) * w.double()


def close(got, ref, dtype, scale=None):
    """|got - ref| <= half a unit of the type at ref + FP32 of the row's (or given) scale."""
    ref = ref.double()
    scale = ref.abs().amax() if scale is None else scale
    err = (got.double() - ref).abs()
    tol = HALF_ULP[dtype] * 1.01 * ref.abs() + FP32 * scale + 1e-37
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_forward(shape, dtype, with_residual, cuda_device):
    x = make(shape, dtype, 1, cuda_device)
    r = make(shape, dtype, 2, cuda_device, 3.0) if with_residual else None
    w = 1 + make(shape[-1:], torch.float32, 3, cuda_device, 0.2)
    y, h = residual_rms_norm(x, w, r)
    assert torch.equal(h, stream_of(x, r))
    ref = norm64(h, w, lnet_b200.norm.RMS_NORM_EPS)
    close(y, ref, dtype, ref.abs())  # every term of the error is relative to the element


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("weight_dtype", DTYPES)
def test_gradient(shape, dtype, weight_dtype, cuda_device):
    if dtype == torch.float32 and weight_dtype == torch.bfloat16:
        pytest.skip("an fp32 stream keeps fp32 weights")
    x = make(shape, dtype, 1, cuda_device).requires_grad_()
    r = make(shape, dtype, 2, cuda_device, 2.0).requires_grad_()
    w = (1 + make(shape[-1:], torch.float32, 3, cuda_device, 0.2)).to(weight_dtype)
    w.requires_grad_()
    dy, dh = make(shape, dtype, 4, cuda_device), make(shape, dtype, 5, cuda_device)
    y, h = residual_rms_norm(x, w, r)
    dx, dr, dw = torch.autograd.grad([y, h], [x, r, w], [dy, dh])
    h64 = h.detach().double().requires_grad_()
    w64 = w.detach().double().requires_grad_()
    y64 = norm64(h64, w64, lnet_b200.norm.RMS_NORM_EPS)
    gh, gw = torch.autograd.grad(y64, [h64, w64], dy.double())
    ref = gh + dh.double()
    # the row's correction term sums products as large as its largest gradient
    close(dx, ref, dtype, (gh.abs().amax(-1, keepdim=True) + dh.double().abs()))
    assert torch.equal(dx, dr)
    xhat = h64.detach() / torch.sqrt((h64.detach() ** 2).mean(-1, keepdim=True)
                                     + lnet_b200.norm.RMS_NORM_EPS)
    mags = (dy.double() * xhat).abs().reshape(-1, shape[-1]).sum(0)
    close(dw, gw, weight_dtype, mags)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 33), (3, 17), (5, 97), (9, 1003), (2, 4100)])
@pytest.mark.parametrize("ahead", [1, 3])
def test_views_off_a_boundary(shape, ahead, dtype, cuda_device):
    """The C ABI on views that start and end inside 16 bytes: what lies around them (NaN) stays out of
    the sums, and the stores inside them."""
    rows, dim = shape
    n, lib = rows * dim, _lib.load()
    kind = 1 if dtype == torch.bfloat16 else 0
    code = torch.cuda.current_stream().cuda_stream

    def view(t=None):
        flat = torch.full((n + 32,), math.nan if t is not None else 77.0, dtype=dtype,
                          device=cuda_device)
        if t is not None:
            flat[ahead:ahead + n] = t.reshape(-1)
        return flat, flat[ahead:ahead + n].view(shape)

    def alone(flat):
        return bool((flat[:ahead] == 77).all()) and bool((flat[ahead + n:] == 77).all())

    x, r, dy, dh = (make(shape, dtype, i, cuda_device) for i in range(1, 5))
    w = 1 + make(shape[-1:], torch.float32, 5, cuda_device, 0.2)
    (_, xv), (_, rv), (_, dyv), (_, dhv) = (view(t) for t in (x, r, dy, dh))
    (yf, y), (hf, h), (dxf, dx) = (view() for _ in range(3))
    rstd = torch.empty(rows, device=cuda_device)
    eps = lnet_b200.norm.RMS_NORM_EPS
    _lib.check(lib.lnet_b200_residual_rms_norm(
        xv.data_ptr(), rv.data_ptr(), w.data_ptr(), kind, 0, rows, dim, eps, y.data_ptr(),
        h.data_ptr(), rstd.data_ptr(), code), "forward")
    assert alone(yf) and alone(hf) and torch.equal(h, stream_of(x, r))
    ref = norm64(h, w, eps)
    close(y, ref, dtype, ref.abs())
    need = ctypes.c_size_t()
    _lib.check(lib.lnet_b200_residual_rms_norm_workspace_size(kind, rows, dim, ctypes.byref(need)),
               "size")
    work, dw = torch.empty(need.value, dtype=torch.uint8, device=cuda_device), torch.empty_like(w)
    # the stream of the view above (its neighbours are 77: finite, and wrong where they count)
    _lib.check(lib.lnet_b200_residual_rms_norm_backward(
        h.data_ptr(), rstd.data_ptr(), w.data_ptr(), dyv.data_ptr(), dhv.data_ptr(), kind, 0, rows,
        dim, dx.data_ptr(), dw.data_ptr(), work.data_ptr(), need.value, code), "backward")
    assert alone(dxf)
    h64, w64 = h.double().requires_grad_(), w.double().requires_grad_()
    gh, gw = torch.autograd.grad(norm64(h64, w64, eps), [h64, w64], dy.double())
    close(dx, gh + dh.double(), dtype, gh.abs().amax(-1, keepdim=True) + dh.double().abs())
    xhat = h.double() / torch.sqrt((h.double() ** 2).mean(-1, keepdim=True) + eps)
    close(dw, gw, torch.float32, (dy.double() * xhat).abs().sum(0))
    codes = torch.full((n + 32,), 77, dtype=torch.uint8, device=cuda_device)
    scales = torch.empty(rows, device=cuda_device)
    want = residual_rms_norm_fp8(x, w, r)
    for at in (ahead, 0):  # the codes' alignment may differ from the rows'
        codes.fill_(77)
        _lib.check(lib.lnet_b200_residual_rms_norm_fp8(
            xv.data_ptr(), rv.data_ptr(), w.data_ptr(), kind, 0, rows, dim, eps,
            codes.data_ptr() + at, scales.data_ptr(), h.data_ptr(), code), "fp8")
        assert alone(hf) and bool((codes[:at] == 77).all()) and bool((codes[at + n:] == 77).all())
        got = codes[at:at + n].view(torch.float8_e4m3fn).view(shape)
        assert torch.allclose(scales, want[1], rtol=1e-5, atol=0)
        # sums of squares taken in another order: a code may round to its neighbour
        near = (got.float() - want[0].float()).abs() <= 2 ** -3 * want[0].float().abs() + 2 ** -9
        assert bool(near.all())


def test_gradient_against_differences(cuda_device):
    x = make((6, 96), torch.float32, 1, cuda_device).requires_grad_()
    w = (1 + make((96,), torch.float32, 2, cuda_device, 0.2)).requires_grad_()
    dy = make((6, 96), torch.float32, 3, cuda_device)
    y, _ = residual_rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    # Central differences of the kernel's own forward: with a step of 1e-2 the cut-off third
    # derivative is ~1e-4 of the slope and rounding 1e-7 / 1e-2 = 1e-5 of the loss.
    step = 1e-2
    for k, (t, grad) in enumerate(((x, dx), (w, dw))):
        v = make(t.shape, torch.float32, 10 + k, cuda_device)

        def loss(s):
            xs = x + s * step * v if t is x else x
            ws = w + s * step * v if t is w else w
            with torch.no_grad():
                return float((residual_rms_norm(xs, ws)[0].double() * dy.double()).sum())

        slope = (loss(1) - loss(-1)) / (2 * step)
        want = float((grad.double() * v.double()).sum())
        assert abs(slope - want) <= 2e-3 * (abs(want) + float(grad.norm() * v.norm()) * 0.1)


def test_gradient_of_one_output_alone(cuda_device):
    x = make((5, 96), torch.float32, 1, cuda_device).requires_grad_()
    r = make((5, 96), torch.float32, 2, cuda_device).requires_grad_()
    w = torch.ones(96, device=cuda_device, requires_grad=True)
    g = make((5, 96), torch.float32, 3, cuda_device)
    y, h = residual_rms_norm(x, w, r)
    only_h = torch.autograd.grad(h, [x, r], g, retain_graph=True)
    assert torch.equal(only_h[0], g) and torch.equal(only_h[1], g)
    dx_y, = torch.autograd.grad(y, [x], g, retain_graph=True)
    dx_both, = torch.autograd.grad([y, h], [x], [g, g])
    assert torch.allclose(dx_both, dx_y + g, rtol=0, atol=1e-6)
    # without a residual the stream is x itself, and both gradients still meet
    y, h = residual_rms_norm(x, w)
    dx, = torch.autograd.grad([y, h], [x], [g, g])
    assert torch.equal(h, x) and dx.shape == x.shape and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_fp8(shape, dtype, cuda_device):
    x, r = make(shape, dtype, 1, cuda_device), make(shape, dtype, 2, cuda_device, 3.0)
    w = 1 + make(shape[-1:], torch.float32, 3, cuda_device, 0.2)
    q, s, h = residual_rms_norm_fp8(x, w, r)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    assert q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(h, stream_of(x, r))
    ref = norm64(h, w, lnet_b200.norm.RMS_NORM_EPS)
    amax = ref.abs().amax(-1)
    assert bool(((s.double() - amax / 448).abs() <= FP32 * amax).all())
    s64 = s.double().unsqueeze(-1)
    err = (q.float().double() * s64 - ref).abs()
    tol = 2.0 ** -4 * ref.abs() + 2.0 ** -10 * s64 + FP32 * ref.abs()
    assert bool((err <= tol).all())
    assert bool((q.float().abs().amax(-1) == 448).all())


def test_special_rows(cuda_device):
    d = 96
    low = torch.finfo(torch.float32).min
    for dtype in DTYPES:
        x = torch.zeros(6, d, dtype=dtype, device=cuda_device)
        x[1, 3] = math.inf
        x[2, 3] = math.nan
        x[3] = 1e-30
        x[4] = -2.0
        x[5, 0] = low if dtype == torch.float32 else torch.finfo(torch.bfloat16).min
        w = torch.ones(d, device=cuda_device)
        y, _ = residual_rms_norm(x, w)
        assert bool((y[0] == 0).all())
        assert bool(y[1, 3].isnan()) and bool((y[1, :3] == 0).all())
        assert bool(y[2].isnan().all())
        assert bool(((y[3].double() - 1e-30 / lnet_b200.norm.RMS_NORM_EPS ** 0.5).abs()
                     <= 1e-2 * 1e-30 / lnet_b200.norm.RMS_NORM_EPS ** 0.5).all())
        assert bool((y[4].float() + 1).abs().max() <= 1e-6)
        assert bool((y[5, 1:] == 0).all())  # the squares overflow: rstd 0, as in the formula
        q, s, _ = residual_rms_norm_fp8(x, w)
        assert bool((q[0].float() == 0).all()) and float(s[0]) == 0
        assert bool(q[2].float().isnan().all()) and bool(s[2].isnan())
        assert float(s[4]) == pytest.approx(1 / 448, rel=1e-5)
        assert bool((q[4].float() == -448).all())


def test_strides_and_alignment(cuda_device):
    base = make((40, 200), torch.bfloat16, 1, cuda_device)
    w = 1 + make((96,), torch.float32, 2, cuda_device, 0.2)
    views = [base[:, 3:99], base[::2, :96], base.t()[:96, :].t().contiguous()[:, :96],
             base.reshape(-1)[5:5 + 96 * 7].reshape(7, 96)]  # rows that start off a 16-byte boundary
    for x in views:
        y, _ = residual_rms_norm(x, w)
        want, _ = residual_rms_norm(x.clone(memory_format=torch.contiguous_format), w)
        close(y, norm64(x, w, lnet_b200.norm.RMS_NORM_EPS), torch.bfloat16)
        assert y.shape == x.shape and want.shape == x.shape


def test_no_rows_and_determinism(cuda_device):
    w = torch.ones(96, device=cuda_device, requires_grad=True)
    x = torch.empty(0, 96, device=cuda_device, requires_grad=True)
    y, h = residual_rms_norm(x, w, x)
    assert y.shape == (0, 96) and h.shape == (0, 96)
    _, dw = torch.autograd.grad(y.sum(), [x, w])
    assert bool((dw == 0).all())
    with torch.no_grad():
        q, s, _ = residual_rms_norm_fp8(x, w, x)
    assert q.shape == (0, 96) and s.shape == (0,)
    x = make((20000, 96), torch.bfloat16, 1, cuda_device).requires_grad_()
    dy = make((20000, 96), torch.bfloat16, 2, cuda_device)
    grads = []
    for _ in range(3):
        y, _ = residual_rms_norm(x, w)
        grads.append(torch.autograd.grad(y, [x, w], dy))
    for g in grads[1:]:
        assert torch.equal(g[0], grads[0][0]) and torch.equal(g[1], grads[0][1])


def test_another_stream(cuda_device):
    x = make((4000, 1024), torch.bfloat16, 1, cuda_device)
    w = torch.ones(1024, device=cuda_device)
    want, _ = residual_rms_norm(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = residual_rms_norm(x, w)
    side.synchronize()
    assert torch.equal(y, want)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 elements: the last rows, forward and backward, against the same rows alone."""
    m, d = (1 << 21) + 100, 1032
    x = torch.ones(m, d, dtype=torch.bfloat16, device=cuda_device)
    x[-64:] = make((64, d), torch.bfloat16, 1, cuda_device)
    w = 1 + make((d,), torch.float32, 2, cuda_device, 0.2)
    x.requires_grad_()
    y, _ = residual_rms_norm(x, w)
    dx, = torch.autograd.grad(y, [x], x.detach())
    tail = x.detach()[-64:].clone().requires_grad_()
    y2, _ = residual_rms_norm(tail, w)
    dx2, = torch.autograd.grad(y2, [tail], tail.detach())
    assert torch.equal(y.detach()[-64:], y2.detach()) and torch.equal(dx[-64:], dx2)


def test_capture(cuda_device):
    """Forward and gradient in a CUDA graph, replayed on new values."""
    x = make((300, 96), torch.bfloat16, 1, cuda_device).requires_grad_()
    w = torch.ones(96, device=cuda_device, requires_grad=True)
    dy = make((300, 96), torch.bfloat16, 2, cuda_device)

    def step():
        y, h = residual_rms_norm(x, w, dy)
        return (y.detach(), *torch.autograd.grad([y, h], [x, w], [dy, dy]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(make((300, 96), torch.bfloat16, 11, cuda_device))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_fp8_refuses_a_gradient(cuda_device):
    x = make((4, 96), torch.bfloat16, 1, cuda_device).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        residual_rms_norm_fp8(x, torch.ones(96, device=cuda_device))


def test_a_second_derivative_is_refused(cuda_device):
    x = make((4, 96), torch.float32, 1, cuda_device).requires_grad_()
    w = torch.ones(96, device=cuda_device, requires_grad=True)
    y, _ = residual_rms_norm(x, w)
    dx, = torch.autograd.grad(y.square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        dx.sum().backward()
