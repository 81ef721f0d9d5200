"""Matrix product with bias, activation and residual, its gradient and its 8-bit form, against the
formula in 64 bits.

Tolerances.  Products of bf16 or e4m3 values are exact in fp32.  A sum of K of them in fp32 has an
error below K 2^-23 of the sum of magnitudes at worst; in any order that adds blocks of 16 at a time
(K / 16 + 16) 2^-23, and the rounding errors of a tensor core's sums (cut, not rounded) all point one
way, so that is taken in full: ACC(K) = (K / 16 + 16) 2^-23 of sum |x w|.  Through f (slope at most
1.13 for GELU and SiLU) it grows by 1.2; exp and erf add a few ulp, 1e-6 of the value.  The result's
rounding is half a unit of bf16, 2^-8 of the value.

The gradient takes its slope from the pre-activation rounded to bf16: an error of 2^-8 |a| |f''(a)|,
and |a f''(a)| <= 0.6 for GELU and SiLU, so 0.6 2^-8 |dy|; its products take da rounded to bf16, 2^-8
|da| an element.  So an element of dx is off by at most 2^-8 (0.6 |dy| + |da|) |W| + ACC, and likewise
dweight and dbias (from the unrounded da: 0.6 2^-8 |dy|).
"""

from __future__ import annotations

import math

import pytest
import torch

from lnet_b200 import linear_act, linear_act_fp8, quantize_rows_fp8

pytestmark = pytest.mark.gpu

HALF = torch.finfo(torch.bfloat16).eps / 2
ACTS = ["none", "relu", "silu", "gelu"]
# rows, inner, outer: one row to the last of the vector kernel, the first of the tiles, sizes on
# both sides of a tile, odd ones (rows off 16 bytes), long k with few tiles (split), many tiles
SHAPES = [(1, 1, 1), (1, 1024, 4096), (2, 96, 384), (3, 1001, 77), (8, 130, 50), (9, 64, 64),
          (127, 96, 129), (128, 128, 128), (129, 72, 257), (300, 1001, 1000), (257, 4096, 96),
          (1000, 40, 1000), (64, 8192, 128), (2048, 512, 2048), (4100, 264, 2056),
          (50, 1, 3), (30, 3, 1), (4, 1003, 9), (300, 72, 1004), (270, 200, 514), (130, 8192, 130),
          (260, 4100, 140)]


def acc(k):
    return (k / 16 + 16) * 2.0 ** -23


def f64(a, act):
    if act == "relu":
        return a.clamp(min=0)
    if act == "silu":
        return a / (1 + torch.exp(-a))
    if act == "gelu":
        return 0.5 * a * (1 + torch.erf(a / math.sqrt(2)))
    return a


def make(shape, seed, device, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).bfloat16().to(device)


def inputs(m, k, n, device, residual=True):
    x, w = make((m, k), 1, device), make((n, k), 2, device, k ** -0.5)
    b = make((n,), 3, device, 0.5)
    return x, w, b, make((m, n), 4, device) if residual else None


def check_forward(y, x, w, b, r, act):
    a = x @ w.t()
    if b is not None:
        a = a + b.double()
    ref = f64(a, act)
    slack = acc(x.shape[1]) * 1.2 * (x.abs() @ w.abs().t()) + 1e-6 * (a.abs() + 1)
    if r is not None:
        ref = ref + r.double()
        slack = slack + 1e-7 * ref.abs()
    err = (y.double() - ref).abs()
    tol = HALF * 1.01 * ref.abs() + slack
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_forward(m, k, n, act, cuda_device):
    x, w, b, r = inputs(m, k, n, cuda_device)
    check_forward(linear_act(x, w, b, r, activation=act), x.double(), w.double(), b, r, act)
    if act in ("none", "gelu"):
        check_forward(linear_act(x, w, activation=act), x.double(), w.double(), None, None, act)


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_gradient(m, k, n, act, cuda_device):
    x, w, b, r = (t.requires_grad_() for t in inputs(m, k, n, cuda_device))
    dy = make((m, n), 5, cuda_device)
    y = linear_act(x, w, b, r, activation=act)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], dy)
    check_forward(y.detach(), x.detach().double(), w.detach().double(), b.detach(), r.detach(),
                  act)
    assert torch.equal(dr, dy)
    x64, w64, b64 = (t.detach().double().requires_grad_() for t in (x, w, b))
    a64 = x64 @ w64.t() + b64
    rx, rw, rb, ra = torch.autograd.grad(f64(a64, act), [x64, w64, b64, a64], dy.double())
    ady = dy.double().abs()
    off = 2.0 ** -8 * 1.05 * (0.6 * (ady if act in ("silu", "gelu") else 0 * ady) + ra.abs())
    if act == "relu":  # a pre-activation that rounds across zero flips its slope
        near = a64.detach().abs() <= acc(k) * (x64.detach().abs() @ w64.detach().abs().t() + 1)
        off = off + near * ady
    ax, aw = x64.detach().abs(), w64.detach().abs()
    for got, ref, slack in (
            (dx, rx, off @ aw + acc(n) * (ra.abs() @ aw)),
            (dw, rw, off.t() @ ax + acc(m) * (ra.abs().t() @ ax)),
            (db, rb, off.sum(0) + 1e-5 * ra.abs().sum(0))):
        err = (got.double() - ref).abs()
        tol = HALF * 1.01 * ref.abs() + slack + 1e-30
        assert bool((err <= tol).all()), float((err - tol).max())


def test_gradient_against_differences(cuda_device):
    """Central differences of the 64-bit loss along the gradients' own inputs."""
    for act in ACTS:
        x, w, b, r = (t.requires_grad_() for t in inputs(40, 64, 72, cuda_device))
        dy = make((40, 72), 5, cuda_device)
        grads = torch.autograd.grad(linear_act(x, w, b, r, activation=act), [x, w, b, r], dy)
        base = [t.detach().double() for t in (x, w, b, r)]
        for i, grad in enumerate(grads):
            v = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i)).double()
            v = v.to(cuda_device)

            def loss(s):
                p = [t + s * 1e-6 * v if j == i else t for j, t in enumerate(base)]
                return float(((f64(p[0] @ p[1].t() + p[2], act) + p[3]) * dy.double()).sum())

            slope = (loss(1) - loss(-1)) / 2e-6
            want = float((grad.double() * v).sum())
            # the gradient's own rounding errors (two of 2^-8 an element at most) against a random
            # direction: four standard deviations of their sum
            assert abs(slope - want) <= 4 * 2 * 2.0 ** -8 * float(grad.double().norm())


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_fp8(m, k, n, act, cuda_device):
    x, w, b, r = inputs(m, k, n, cuda_device)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    y = linear_act_fp8(xq, xs, wq, ws, b, r, activation=act)
    xd = xq.double() * xs.double().unsqueeze(-1)
    wd = wq.double() * ws.double().unsqueeze(-1)
    check_forward(y, xd, wd, b, r, act)


def test_quantize_rows(cuda_device):
    for dtype in (torch.float32, torch.bfloat16):
        t = make((7, 333), 1, cuda_device).to(dtype)
        t[3] = 0
        q, s = quantize_rows_fp8(t)
        amax = t.double().abs().amax(-1)
        assert bool(((s.double() - amax / 448).abs() <= 1e-6 * amax).all())
        assert float(s[3]) == 0 and bool((q[3].float() == 0).all())
        err = (q.double() * s.double().unsqueeze(-1) - t.double()).abs()
        tol = 2.0 ** -4 * t.double().abs() + (2.0 ** -10 + 1e-6) * s.double().unsqueeze(-1)
        assert bool((err <= tol * 1.0001).all())


def test_strides_alignment_and_shapes(cuda_device):
    x, w, b, r = inputs(60, 96, 80, cuda_device)
    wide = torch.zeros(60, 200, dtype=x.dtype, device=cuda_device)
    wide[:, 3:99] = x
    flat = torch.zeros(60 * 96 + 1, dtype=x.dtype, device=cuda_device)
    flat[1:] = x.reshape(-1)
    want = linear_act(x, w, b, r, activation="silu")
    for view in (wide[:, 3:99], flat[1:].reshape(60, 96), x.t().contiguous().t()):
        assert torch.equal(linear_act(view, w, b, r, activation="silu"), want)
    wt = w.t().contiguous().t()
    assert torch.equal(linear_act(x, wt, b, r.t().contiguous().t(), activation="silu"), want)
    y = linear_act(x.reshape(3, 20, 96), w, b, r.reshape(3, 20, 80), activation="silu")
    assert y.shape == (3, 20, 80) and torch.equal(y.reshape(60, 80), want)
    one = linear_act(x[0], w, b, r[0], activation="silu")
    assert one.shape == (80,)
    # an output row pitch that keeps no 16-byte alignment, and a bias off it
    odd_bias = torch.cat([b[:1], b])[1:]
    assert torch.equal(linear_act(x, w, odd_bias, r, activation="silu"), want)


def test_rows_further_apart_than_their_length(cuda_device):
    """Operands with a row pitch are read as they lie, forward and backward, few rows and many."""
    for m in (5, 60, 300):
        x, w, b, r = inputs(m, 96, 80, cuda_device)
        wide_x = torch.full((m, 200), math.nan, dtype=x.dtype, device=cuda_device)
        wide_w = torch.full((80, 136), math.nan, dtype=x.dtype, device=cuda_device)
        wide_x[:, 8:104], wide_w[:, 16:112] = x, w
        dy = make((m, 80), 5, cuda_device)
        grads = []
        for xi, wi in ((x, w), (wide_x[:, 8:104], wide_w[:, 16:112])):
            xi, wi = xi.detach().requires_grad_(), wi.detach().requires_grad_()
            y = linear_act(xi, wi, b, r, activation="gelu")
            grads.append((y.detach(), *torch.autograd.grad(y, [xi, wi], dy)))
        assert all(torch.equal(p, q) for p, q in zip(*grads))
        xq, xs = quantize_rows_fp8(x)
        wq, ws = quantize_rows_fp8(w)
        want = linear_act_fp8(xq, xs, wq, ws, b, r)
        pad = torch.zeros(m, 160, dtype=torch.uint8, device=cuda_device)
        pad[:, 16:112] = xq.view(torch.uint8)
        assert torch.equal(linear_act_fp8(pad.view(xq.dtype)[:, 16:112], xs, wq, ws, b, r), want)


def test_infinities_stay_in_their_rows(cuda_device):
    x, w, b, _ = inputs(200, 96, 160, cuda_device)
    x[17, 5] = math.inf
    x[130, 7] = math.nan
    y = linear_act(x, w, b)
    bad = torch.zeros(200, dtype=torch.bool, device=cuda_device)
    bad[17] = bad[130] = True
    assert torch.equal((~torch.isfinite(y)).any(-1), bad)


def test_no_rows_and_partial_gradients(cuda_device):
    x, w, b, r = inputs(0, 96, 80, cuda_device)
    w.requires_grad_(), b.requires_grad_()
    y = linear_act(x, w, b, r, activation="gelu")
    assert y.shape == (0, 80)
    dw, db = torch.autograd.grad(y.sum(), [w, b])
    assert bool((dw == 0).all()) and bool((db == 0).all())
    x, w, b, r = inputs(70, 96, 80, cuda_device)
    dy = make((70, 80), 5, cuda_device)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear_act(*full, activation="gelu"), full, dy)
    for i in range(4):
        ts = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b, r))]
        g, = torch.autograd.grad(linear_act(*ts, activation="gelu"), [ts[i]], dy)
        assert torch.equal(g, grads[i])


def test_determinism_and_streams(cuda_device):
    x, w, b, r = (t.requires_grad_() for t in inputs(3000, 96, 384, cuda_device))
    dy = make((3000, 384), 5, cuda_device)

    def step():
        y = linear_act(x, w, b, r, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, [x, w, b, r], dy))

    first = step()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_capture(cuda_device):
    """Forward and gradient in a CUDA graph, replayed on new values."""
    x, w, b, r = (t.requires_grad_() for t in inputs(300, 96, 384, cuda_device))
    dy = make((300, 384), 5, cuda_device)

    def step():
        y = linear_act(x, w, b, r, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(make((300, 96), 11, cuda_device))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_offsets_past_32_bits(cuda_device):
    """An output of more than 2^31 elements: its last rows against the same rows alone."""
    m, k, n = (1 << 21) + 300, 64, 1032
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda_device)
    x[-200:] = make((200, k), 1, cuda_device)
    w, b = make((n, k), 2, cuda_device), make((n,), 3, cuda_device)
    y = linear_act(x, w, b, activation="relu")
    assert y.numel() > 1 << 31
    assert torch.equal(y[-200:], linear_act(x[-200:].clone(), w, b, activation="relu"))
    assert torch.equal(y[:100], linear_act(x[:100].clone(), w, b, activation="relu"))


def test_fp8_refuses_a_gradient(cuda_device):
    x, w, b, _ = inputs(4, 96, 80, cuda_device)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_act_fp8(xq, xs, wq, ws, b.requires_grad_())
