"""8-bit rows (``quantize_rows_fp8``, ``residual_rms_norm_fp8``) of ordinary, tiny and subnormal values
against the definition: scale = max|y| / 448, code = e4m3(y / scale), a row whose scale is 0 all zeros.

Tolerances.  A scale that is a quotient of fp32 numbers is exact to its rounding, 2^-24 of it or, below the
normals, 2^-150.  A code is off by half a step (2^-4 of the value, 2^-10 of the scale below e4m3's normals)
and by a few fp32 roundings before it (FP32 of the value).  A scale rounded below the normals may leave
values above 448 scales, which saturate.  The norm's y has FP32 of itself and two roundings of 2^-150.
"""

from __future__ import annotations

import pytest
import torch

import lnet_b200
from lnet_b200 import linear_act_fp8, quantize_rows_fp8, residual_rms_norm_fp8

pytestmark = pytest.mark.gpu

FP32 = 4e-6
UNIT = 2.0 ** -149  # the smallest subnormal
DTYPES = [torch.float32, torch.bfloat16]
# largest magnitudes: ordinary, on both sides of 448 / FLT_MAX = 1.32e-36, scales around the smallest
# normal number, subnormal scales, a scale of one unit, a scale that rounds to 0
LARGEST = [1.0, 1e-30, 1.4e-36, 1.2e-36, 1e-37, 1e-38, 1e-40, 1e-42, 3.2e-43, 3e-44]


def pattern(rows, dim, device):
    """Values in [-1, 1] in 64 bits with exact zeros among them, the largest magnitude 1."""
    g = torch.Generator().manual_seed(rows + dim)
    t = torch.rand(rows, dim, generator=g, dtype=torch.float64) * 2 - 1
    t[torch.rand(rows, dim, generator=g) < 0.3] = 0
    t[:, dim // 2] = -1
    return t.to(device)


def check_codes(q, s, y64, slack):
    """`slack`: what y itself may be off by."""
    assert bool(torch.isfinite(q.float()).all())
    s64, q64 = s.double().unsqueeze(-1), q.float().double()
    tol = 2.0 ** -4 * y64.abs() + 2.0 ** -10 * s64 + slack + (y64.abs() - 448 * s64).clamp(min=0)
    live = (s64 > 0).expand_as(q64)
    err = (q64 * s64 - y64).abs()
    assert bool((err <= tol)[live].all()), float((err - tol)[live].max())
    assert bool((q64[~live] == 0).all())
    assert bool((q64[y64 == 0] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 5, 33, 64, 96, 333, 4096, 4097, 20001])
def test_quantized_rows(dim, dtype, cuda_device):
    big = torch.tensor(LARGEST, dtype=torch.float64, device=cuda_device).unsqueeze(-1)
    t = (pattern(len(LARGEST), dim, cuda_device) * big).float().to(dtype)
    q, s = quantize_rows_fp8(t)
    y64 = t.double()
    amax = y64.abs().amax(-1)
    assert bool(((s.double() - amax / 448).abs() <= 2.0 ** -24 * amax / 448 + UNIT / 2).all())
    check_codes(q, s, y64, FP32 * y64.abs())
    ordinary = slice(0, 6)  # scales of full precision: the largest element is the largest code
    assert bool((q[ordinary].float().abs().amax(-1) == 448).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [5, 33, 96, 4096, 20001])
@pytest.mark.parametrize("largest", LARGEST)
def test_normed_rows(largest, dim, dtype, cuda_device):
    # |x| <= 1e-32 leaves rstd = eps^-1/2 = 2896, and the weight takes y to its magnitude
    x = (pattern(7, dim, cuda_device) * 1e-32).float().to(dtype)
    eps = lnet_b200.norm.RMS_NORM_EPS
    unit = float(x.double().abs().max()) / eps ** 0.5
    w = torch.full((dim,), largest / unit, dtype=torch.float64, device=cuda_device).float()
    q, s, _ = residual_rms_norm_fp8(x, w)
    x64 = x.double()
    y64 = x64 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps) * w.double()
    amax = y64.abs().amax(-1)
    assert bool(((s.double() - amax / 448).abs() <= FP32 * amax / 448 + 2 * UNIT).all())
    check_codes(q, s, y64, FP32 * y64.abs() + 2 * UNIT)


def test_a_tiny_weight_row_stays_in_its_column(cuda_device):
    """A row of weights that decayed to 1e-37, with zeros: its column of the product is about 0, not NaN."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(64, 96, generator=g)
    w[5] *= 1e-37
    w[5, ::3] = 0
    x = torch.randn(20, 96, generator=g)
    wq, ws = quantize_rows_fp8(w.to(cuda_device))
    xq, xs = quantize_rows_fp8(x.to(cuda_device))
    y = linear_act_fp8(xq, xs, wq, ws).float()
    assert bool(torch.isfinite(y).all()) and float(y[:, 5].abs().max()) < 1e-34
    assert float(y.abs().max()) > 1


@pytest.mark.parametrize("dim", [64, 4096, 1001])
def test_rows_with_infinities_and_nan(dim, cuda_device):
    for dtype in DTYPES:
        t = torch.ones(4, dim, dtype=dtype, device=cuda_device)
        t[1, 3], t[2, 3], t[3] = float("inf"), float("nan"), 0
        q, s = quantize_rows_fp8(t)
        assert float(s[0]) == pytest.approx(1 / 448, rel=1e-6) and bool((q[0].float() == 448).all())
        assert float(s[1]) == float("inf")
        assert bool(q[1, 3].float().isnan()) and bool((q[1, 4:].float() == 0).all())
        assert bool(s[2].isnan()) and bool(q[2].float().isnan().all())
        assert float(s[3]) == 0 and bool((q[3].float() == 0).all())
