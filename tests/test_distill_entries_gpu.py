"""Distillation with many entries a row; tolerances of test_distill_gpu."""

from __future__ import annotations

import math

import pytest
import torch
from test_distill_gpu import DTYPES, check, make

from lnet_b200 import distillation_loss

pytestmark = pytest.mark.gpu


# entries on both sides of the sizes where the kernels change, a teacher whose whole distribution was
# kept, few rows (several blocks a row) and many
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,top", [(5, 1000, 256), (5, 1000, 257), (5, 1000, 1000),
                                              (4, 4099, 4099), (3, 9001, 5000), (2, 100003, 1000),
                                              (2, 70001, 20000), (200, 5003, 700)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_many_entries(rows, classes, top, dtype, reduction, cuda_device):
    z, index, teacher, labels = make(rows, classes, top, dtype, rows + classes, cuda_device)
    check(z, index, teacher, labels, 2.0, 0.6, reduction, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes", [(5, 700), (3, 30011), (1, 100003)])
def test_many_duplicates(rows, classes, dtype, cuda_device):
    """Entries that name a class several times add up, the label's among them; padding between them."""
    g = torch.Generator().manual_seed(classes)
    z = (torch.randn(rows, classes, generator=g) * 2).to(dtype).to(cuda_device)
    index = torch.randint(0, min(classes, 9000), (rows, 3001), generator=g)
    index[:, ::7] = index[:, :1]
    index[:, 5::11] = -1
    teacher = torch.randn(rows, 3001, generator=g)
    teacher[:, 3::13] = -math.inf
    labels = index[:, 0].clone()
    check(z, index.to(cuda_device), teacher.to(cuda_device), labels.to(cuda_device), 1.5, 0.7, "mean",
          dtype)


def test_many_entries_give_the_same_bits_every_time(cuda_device):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(40, 3000, generator=g).to(cuda_device).requires_grad_()
    index = torch.randint(0, 50, (40, 2000), generator=g).to(cuda_device)
    teacher = torch.randn(40, 2000, generator=g).to(cuda_device)
    runs = [torch.autograd.grad(distillation_loss(z, index, teacher), z)[0] for _ in range(4)]
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_the_work_grows_with_the_entries_and_not_with_their_square(cuda_device):
    g = torch.Generator().manual_seed(1)
    rows, classes = 296, 32768
    z = torch.randn(rows, classes, generator=g).bfloat16().to(cuda_device).requires_grad_()
    order = torch.randperm(classes, generator=g)

    def milliseconds(top):
        index = order[:top].expand(rows, top).contiguous().to(cuda_device)
        teacher = torch.randn(rows, top, generator=g).to(cuda_device)
        times = []
        for _ in range(4):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            torch.autograd.grad(distillation_loss(z, index, teacher), z)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times[1:])

    # four times the entries: about four times the time, where the square would take 16
    assert milliseconds(16384) <= 8 * milliseconds(4096)
