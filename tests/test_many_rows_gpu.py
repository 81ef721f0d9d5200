"""The norm and the linear over more rows than a wave of blocks or tiles, as the image workload's streams
have them; the checks and tolerances of their own tests."""

from __future__ import annotations

import pytest
import test_linear_gpu as linear
import test_norm_gpu as norm
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,dtype", [((256, 784, 96), torch.bfloat16), ((50021, 97), torch.float32),
                                         ((70001, 200), torch.bfloat16), ((100003, 24), torch.float32)])
def test_norm(shape, dtype, cuda_device):
    norm.test_forward(shape, dtype, True, cuda_device)
    norm.test_gradient(shape, dtype, torch.float32, cuda_device)
    norm.test_fp8(shape, dtype, cuda_device)


@pytest.mark.parametrize("m,k,n,act", [(50176, 96, 384, "gelu"), (50176, 384, 96, "none"),
                                       (20011, 96, 130, "silu"), (33001, 40, 100, "relu")])
def test_linear(m, k, n, act, cuda_device):
    linear.test_gradient(m, k, n, act, cuda_device)
