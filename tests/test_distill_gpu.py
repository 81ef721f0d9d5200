"""The distillation loss and its gradient against the formula in 64 bits.

Tolerances.  log q and the softmax come from an fp32 sum of V exponentials (ex2.approx, 2 ulp) whose
arguments (z - m) / tau are rounded once: a relative error of 2^-24 |z - m| log2(e) / tau + 2^-22 for
each term.  The cases have |z - m| <= 40, so 40 * 1.45 * 2^-24 + 2^-22 = 3.7e-6; FP32 = 8e-6 covers
the sum and the division too.  A loss is a sum of terms p (log p - log q) of up to 40: an absolute
error of FP32 (its magnitude + 1).  A bf16 gradient adds half a unit in the last place, 2^-8 of
the value (8 significant bits).
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lnet_b200 import _lib, distillation_loss

pytestmark = pytest.mark.gpu

FP32 = 8e-6
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}
DTYPES = [torch.float32, torch.bfloat16]


def reference(z, index, teacher, labels, tau, alpha, reduction):
    """Loss in 64 bits from the definition, row by row."""
    losses, counted = [], 0
    z = z.double()
    for i in range(z.shape[0]):
        keep = (index[i] >= 0) & (teacher[i] > -math.inf)
        loss = z[i].sum() * 0 if bool(torch.isfinite(z[i]).all()) else z.new_zeros(())
        if bool(keep.any()):
            t = teacher[i][keep].double() / tau
            p = torch.softmax(t, -1)
            logq = torch.log_softmax(z[i] / tau, -1)[index[i][keep]]
            kl = (torch.xlogy(p, p) - torch.where(p > 0, p * logq, torch.zeros_like(p))).sum()
            loss = loss + alpha * tau * tau * kl
        has = labels is not None and int(labels[i]) >= 0
        if has and alpha != 1:
            loss = loss - (1 - alpha) * torch.log_softmax(z[i], -1)[labels[i]]
        counted += bool(keep.any()) or has
        losses.append(loss)
    losses = torch.stack(losses)
    if reduction == "none":
        return losses
    return losses.sum() / (max(counted, 1) if reduction == "mean" else 1)


def make(rows, classes, top, dtype, seed, device, labels=True, masked=0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, classes, generator=g) * 2
    t = z * 0.7 + torch.randn(rows, classes, generator=g)
    if masked:
        off = torch.randperm(classes, generator=g)[:masked]
        z[:, off] = -math.inf
        t[:, off] = -math.inf
    kept, index = torch.topk(t, top, -1)
    if rows > 1:
        index[1, top // 2:] = -1  # a ragged row
    if rows > 2:
        index[2] = -1  # a row without the teacher
    lab = index[:, 0].clamp(min=0).clone()
    if rows > 3:
        lab[3] = -100
    return (z.to(dtype).to(device), index.to(device), kept.to(device),
            lab.to(device) if labels else None)


def check(z, index, teacher, labels, tau, alpha, reduction, dtype):
    zg = z.clone().requires_grad_()
    loss = distillation_loss(zg, index, teacher, labels=labels, temperature=tau, alpha=alpha,
                             reduction=reduction)
    assert loss.dtype == torch.float32
    up = torch.linspace(0.5, 2.0, loss.numel(), device=z.device).reshape(loss.shape)
    if reduction != "none":
        up = torch.full((), 1.0, device=z.device)
    dz, = torch.autograd.grad(loss, zg, up)
    z64 = z.double().requires_grad_()
    ref = reference(z64, index, teacher, labels, tau, alpha, reduction)
    ref_dz, = torch.autograd.grad(ref, z64, up.double())
    # 0 * -inf of autograd's own chain at masked classes: their gradient is 0
    ref_dz = torch.where(torch.isinf(z), torch.zeros_like(ref_dz), ref_dz)
    err = (loss.double() - ref).abs()
    assert bool((err <= FP32 * tau * tau * (ref.abs() + 1)).all()), float(err.max())
    err = (dz.double() - ref_dz).abs()
    # each entry is a difference of probabilities of at most the row's largest weight
    unit = (alpha * tau + 1) * (up.reshape(-1, 1).double() if reduction == "none" else 1.0)
    if reduction == "mean":
        keep = ((index >= 0) & (teacher > -math.inf)).any(-1)
        n = (keep | (labels >= 0) if labels is not None else keep).sum()
        unit = unit / max(int(n), 1)
    tol = HALF_ULP[dtype] * 1.01 * ref_dz.abs() + FP32 * unit
    assert bool((err <= tol).all()), float((err - tol).max())


# classes: one, a few, odd ones, a cluster's worth in one row, more than a block holds at once
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (5, 3, 2), (4, 10, 4), (37, 1000, 10),
                                              (6, 1001, 7), (9, 4099, 33), (300, 517, 5),
                                              (3, 70001, 16), (5, 32768, 64), (1, 100003, 40),
                                              (700, 4099, 80), (250, 8200, 200), (3, 9000, 300)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_and_gradient(rows, classes, top, dtype, reduction, cuda_device):
    z, index, teacher, labels = make(rows, classes, top, dtype, rows + classes, cuda_device)
    check(z, index, teacher, labels, 2.0, 0.6, reduction, dtype)


# rows that 2 to 8 blocks share (8192 bf16 or 4096 fp32 classes each), whole and with a block of little
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [8191, 8193, 12001, 16385, 20001, 24576, 28673, 32767, 40003,
                                     50257, 57344, 65535])
def test_rows_of_several_blocks(classes, dtype, cuda_device):
    z, index, teacher, labels = make(5, classes, 24, dtype, classes, cuda_device)
    check(z, index, teacher, labels, 2.0, 0.6, "mean", dtype)
    check(z, index, teacher, labels, 1.0, 0.6, "sum", dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (3, 3, 2), (1, 7, 3), (5, 9, 4), (4, 1003, 5),
                                              (3, 8190, 6), (2, 20005, 30)])
@pytest.mark.parametrize("ahead", [1, 3])
def test_logits_and_gradient_off_a_boundary(rows, classes, top, ahead, dtype, cuda_device):
    """The C ABI on a view that starts and ends inside 16 bytes: what lies around it stays out of the
    loss (it is NaN) and of the gradient's stores."""
    z, index, teacher, labels = make(rows, classes, top, dtype, classes + ahead, cuda_device)
    n = rows * classes
    flat = torch.full((n + 32,), math.nan, dtype=dtype, device=cuda_device)
    flat[ahead:ahead + n] = z.reshape(-1)
    grad = torch.full((n + 32,), 77.0, dtype=dtype, device=cuda_device)
    size = flat.element_size()
    q = _lib.DistillRequest(rows, classes, top, 1 if dtype == torch.bfloat16 else 0, 1,
                            flat.data_ptr() + ahead * size, index.data_ptr(), teacher.data_ptr(),
                            labels.data_ptr(), 2.0, 0.6)
    lib, need = _lib.load(), ctypes.c_size_t()
    _lib.check(lib.lnet_b200_distill_workspace_size(ctypes.byref(q), ctypes.byref(need)), "size")
    work = torch.empty(need.value, dtype=torch.uint8, device=cuda_device)
    loss = torch.empty((), device=cuda_device)
    _lib.check(lib.lnet_b200_distill_forward(
        ctypes.byref(q), work.data_ptr(), need.value, loss.data_ptr(),
        grad.data_ptr() + ahead * size, torch.cuda.current_stream().cuda_stream), "forward")
    assert bool((grad[:ahead] == 77).all()) and bool((grad[ahead + n:] == 77).all())
    zg = z.clone().requires_grad_()
    want = distillation_loss(zg, index, teacher, labels=labels, temperature=2.0, alpha=0.6,
                             reduction="sum")
    dz, = torch.autograd.grad(want, zg)
    assert float((loss - want.detach()).abs()) <= 2 * FP32 * 4.0 * (rows + float(want.detach().abs()))
    tol = 2 * HALF_ULP[dtype] * 1.01 * dz.double().abs() + 2 * FP32 * 2.2
    assert bool(((grad[ahead:ahead + n].double().view_as(dz) - dz.double()).abs() <= tol).all())


@pytest.mark.parametrize("tau,alpha,labelled", [(1.0, 1.0, False), (1.0, 0.5, True),
                                                (4.0, 1.0, True), (1.5, 0.9, True),
                                                (3.0, 0.0, True), (0.5, 0.3, True)])
@pytest.mark.parametrize("masked", [0, 300])
def test_temperatures_and_masks(tau, alpha, labelled, masked, cuda_device):
    z, index, teacher, labels = make(17, 2003, 12, torch.float32, 5, cuda_device, labelled, masked)
    check(z, index, teacher, labels, tau, alpha, "mean", torch.float32)


def test_gradient_against_differences(cuda_device):
    z, index, teacher, labels = make(5, 50, 6, torch.float32, 9, cuda_device)
    kw = dict(labels=labels, temperature=2.0, alpha=0.7)
    zg = z.clone().requires_grad_()
    dz, = torch.autograd.grad(distillation_loss(zg, index, teacher, **kw), zg)
    v = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).to(z.device)
    step = 1e-2  # third derivatives of a softmax are below 1: 1e-4 of the slope; rounding 1e-5
    up, down = (float(distillation_loss(z + s * step * v, index, teacher, **kw)) for s in (1, -1))
    want = float((dz.double() * v.double()).sum())
    assert abs((up - down) / (2 * step) - want) <= 2e-3 * (abs(want) + float(dz.norm()))


def test_scaled_and_repeated_backward(cuda_device):
    for reduction in ("mean", "none"):
        z, index, teacher, labels = make(8, 1000, 10, torch.float32, 3, cuda_device)
        z.requires_grad_()
        loss = distillation_loss(z, index, teacher, labels=labels, temperature=2.0, alpha=0.5,
                                 reduction=reduction).sum()
        first, = torch.autograd.grad(loss, z, retain_graph=True)
        first = first.clone()
        second, = torch.autograd.grad(3 * loss, z, retain_graph=True)
        third, = torch.autograd.grad(loss, z)
        scale = float(first.abs().max())
        assert float((second - 3 * first).abs().max()) <= 1e-6 * 3 * scale
        assert float((third - first).abs().max()) <= 1e-6 * scale
        assert torch.equal(torch.autograd.grad(
            distillation_loss(z, index, teacher, labels=labels, temperature=2.0, alpha=0.5,
                              reduction=reduction).sum() * 0.25, z)[0] * 4, third) or \
            float((third - first).abs().max()) <= 1e-6 * scale


def test_duplicate_entries(cuda_device):
    z, _, _, _ = make(2, 40, 4, torch.float32, 3, cuda_device)
    index = torch.tensor([[3, 7, 3, 9], [5, 5, 5, 5]], device=cuda_device)
    teacher = torch.tensor([[1.0, 2.0, 0.5, -1.0], [0.0, 1.0, 2.0, 3.0]], device=cuda_device)
    labels = torch.tensor([3, 39], device=cuda_device)
    check(z, index, teacher, labels, 2.0, 0.5, "mean", torch.float32)


def test_rows_that_leave_nothing(cuda_device):
    inf = math.inf
    z = torch.zeros(6, 20, device=cuda_device)
    z[1] = -inf          # nothing left, and no target
    z[2] = -inf          # nothing left, with a target
    z[3, 4] = -inf       # the teacher's mass on a masked class
    z[4] = torch.finfo(torch.float32).min  # masked by the type's lowest value: uniform
    index = torch.tensor([[1, 2], [-1, -1], [3, 4], [4, 5], [0, 1], [6, 7]], device=cuda_device)
    teacher = torch.zeros(6, 2, device=cuda_device)
    teacher[5] = -inf    # entries without mass are padding
    z.requires_grad_()
    loss = distillation_loss(z, index, teacher, reduction="none")
    dz, = torch.autograd.grad(loss, z, torch.ones(6, device=cuda_device))
    loss = loss.detach()
    kl = math.log(20) - math.log(2)
    assert float(loss[0]) == pytest.approx(kl, rel=1e-5)
    assert float(loss[1]) == 0 and bool((dz[1] == 0).all())
    assert float(loss[2]) == inf and float(loss[3]) == inf
    want = torch.zeros(20, device=cuda_device)
    want[3:5] = -0.5
    assert torch.allclose(dz[2], want)
    assert float(dz[3, 4]) == pytest.approx(-0.5) and float(dz[3, 0]) == pytest.approx(1 / 19)
    assert float(loss[4]) == pytest.approx(kl, rel=1e-5)
    assert float(loss[5]) == 0 and bool((dz[5] == 0).all())
    # the same rows through the kernels that take loss and gradient together
    ok = torch.tensor([0, 1, 4, 5], device=cuda_device)
    z3 = z.detach()[ok].clone().requires_grad_()
    total = distillation_loss(z3, index[ok], teacher[ok], reduction="sum")
    assert float(total.detach()) == pytest.approx(2 * kl, rel=1e-5)
    assert torch.allclose(torch.autograd.grad(total, z3)[0], dz[ok])
    for i in (2, 3):
        zi = z.detach()[i:i + 1].clone().requires_grad_()
        total = distillation_loss(zi, index[i:i + 1], teacher[i:i + 1], reduction="sum")
        assert float(total.detach()) == inf
        assert torch.allclose(torch.autograd.grad(total, zi)[0], dz[i:i + 1])
    none = torch.full((6, 2), -1, device=cuda_device)
    z2 = z.detach().clone().requires_grad_()
    total = distillation_loss(z2, none, teacher)
    grad, = torch.autograd.grad(total, z2)
    assert float(total.detach()) == 0 and bool((grad == 0).all())


def test_infinite_and_nan_logits(cuda_device):
    z = torch.zeros(3, 8, device=cuda_device)
    z[0, 1], z[1, 2] = math.inf, math.nan
    index = torch.zeros(3, 1, dtype=torch.int64, device=cuda_device)
    loss = distillation_loss(z, index, torch.zeros(3, 1, device=cuda_device), reduction="none")
    assert bool(loss[:2].isnan().all()) and float(loss[2]) == pytest.approx(math.log(8), rel=1e-5)
    z.requires_grad_()
    total = distillation_loss(z, index, torch.zeros(3, 1, device=cuda_device))
    dz, = torch.autograd.grad(total, z)
    assert bool(total.isnan()) and bool(dz[:2].isnan().all()) and bool(torch.isfinite(dz[2]).all())


def test_an_index_past_the_classes_is_nan_and_stays_in_its_row(cuda_device):
    z, index, teacher, labels = make(6, 100, 4, torch.float32, 3, cuda_device)
    index[0, 1] = 100
    labels[4] = 1 << 40
    z.requires_grad_()
    loss = distillation_loss(z, index, teacher, labels=labels, alpha=0.5, reduction="none")
    dz, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    bad = torch.tensor([True, False, False, False, True, False], device=cuda_device)
    assert torch.equal(loss.isnan(), bad)
    assert torch.equal(dz.isnan().all(-1), bad) and torch.equal(dz.isnan().any(-1), bad)


def test_shapes_strides_and_streams(cuda_device):
    z, index, teacher, labels = make(12, 777, 5, torch.bfloat16, 3, cuda_device)
    kw = dict(temperature=2.0, alpha=0.5, reduction="none")
    want = distillation_loss(z, index, teacher, labels=labels, **kw)
    wide = torch.empty(12, 1000, dtype=z.dtype, device=cuda_device)
    wide[:, 3:780] = z
    got = distillation_loss(wide[:, 3:780], index.t().contiguous().t(), teacher.bfloat16().float(),
                            labels=labels, **kw)
    assert got.shape == (12,)
    got = distillation_loss(z.reshape(3, 4, 777), index.reshape(3, 4, 5),
                            teacher.reshape(3, 4, 5), labels=labels.reshape(3, 4), **kw)
    assert torch.equal(got.reshape(-1), want)
    flat = torch.empty(12 * 777 + 1, dtype=z.dtype, device=cuda_device)
    flat[1:] = z.reshape(-1)
    odd = flat[1:].reshape(12, 777).requires_grad_()  # starts off a 16-byte boundary
    loss = distillation_loss(odd, index, teacher, labels=labels, temperature=2.0, alpha=0.5)
    g1, = torch.autograd.grad(loss, odd)
    z.requires_grad_()
    loss = distillation_loss(z, index, teacher, labels=labels, temperature=2.0, alpha=0.5)
    g2, = torch.autograd.grad(loss, z)
    assert float((g1.float() - g2.float()).abs().max()) <= 2 ** -8 * float(g2.float().abs().max())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        got = distillation_loss(z, index, teacher, labels=labels, **kw)
    side.synchronize()
    assert torch.equal(got, want)


def test_no_rows_no_entries_and_determinism(cuda_device):
    z = torch.zeros(0, 10, device=cuda_device)
    index = torch.zeros(0, 3, dtype=torch.int64, device=cuda_device)
    assert float(distillation_loss(z, index, torch.zeros(0, 3, device=cuda_device))) == 0
    z, index, teacher, labels = make(8, 100, 4, torch.float32, 3, cuda_device)
    loss = distillation_loss(z, index[:, :0], teacher[:, :0], labels=labels, alpha=0.0)
    ref = reference(z, index[:, :0], teacher[:, :0], labels, 1.0, 0.0, "mean")
    assert float(loss) == pytest.approx(float(ref), rel=1e-5)
    check(z, index[:, :0], teacher[:, :0], labels, 1.0, 0.0, "mean", torch.float32)
    z, index, teacher, labels = make(500, 1000, 10, torch.bfloat16, 3, cuda_device)
    z.requires_grad_()
    runs = []
    for _ in range(3):
        loss = distillation_loss(z, index, teacher, labels=labels, temperature=2.0, alpha=0.5)
        runs.append((loss.detach(), torch.autograd.grad(loss, z)[0]))
    assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1]) for r in runs)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 logits: the last rows' losses and gradients against the same rows alone."""
    rows, classes = 32800, 65504
    z = torch.zeros(rows, classes, dtype=torch.bfloat16, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    z[-8:] = (torch.randn(8, classes, generator=g) * 2).bfloat16().to(cuda_device)
    index = torch.randint(0, classes, (rows, 4), generator=g).to(cuda_device)
    teacher = torch.randn(rows, 4, generator=g).to(cuda_device)
    z.requires_grad_()
    loss = distillation_loss(z, index, teacher, reduction="sum")
    dz, = torch.autograd.grad(loss, z)
    tail = z.detach()[-8:].clone().requires_grad_()
    loss2 = distillation_loss(tail, index[-8:], teacher[-8:], reduction="sum")
    dz2, = torch.autograd.grad(loss2, tail)
    assert z.numel() > 1 << 31 and torch.equal(dz[-8:], dz2)
    each = distillation_loss(z.detach(), index, teacher, reduction="none")
    assert torch.equal(each[-8:], distillation_loss(tail.detach(), index[-8:], teacher[-8:],
                                                    reduction="none")) or \
        float((each[-8:].sum() - loss2.detach()).abs()) <= 1e-4 * float(loss2.detach())
    assert float((each.double().sum() - loss.detach().double()).abs()) <= 1e-5 * float(loss.detach())


def test_capture(cuda_device):
    """Loss and gradient in a CUDA graph, replayed on new logits."""
    z, index, teacher, labels = make(40, 1000, 10, torch.float32, 3, cuda_device)
    z.requires_grad_()

    def step():
        loss = distillation_loss(z, index, teacher, labels=labels, temperature=2.0, alpha=0.5)
        return loss.detach(), torch.autograd.grad(loss, z)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        z.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, step()))
