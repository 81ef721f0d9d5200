"""The 8-bit feed-forward block over a module's life: new weights, moves, and inputs that want a gradient."""

from __future__ import annotations

import copy

import pytest
import torch

from lnet_b200 import B200FeedForward

pytestmark = pytest.mark.gpu


def make(seed, device):
    torch.manual_seed(seed)
    block = B200FeedForward(96, 384, device=device)
    with torch.no_grad():
        block.norm_weight.uniform_(0.5, 1.5)
    return block


def tokens(device):
    g = torch.Generator().manual_seed(7)
    return torch.randn(50, 96, generator=g).bfloat16().to(device)


def fresh(block, device):
    """What a block quantised only now gives."""
    new = B200FeedForward(96, 384, device=device)
    new.load_state_dict(block.state_dict())
    return new.quantize_()


def test_weights_that_change_after_quantize(cuda_device):
    x = tokens(cuda_device)
    block, other = make(1, cuda_device).quantize_(), make(2, cuda_device)
    before = block(x)
    block.load_state_dict(other.state_dict())
    assert torch.equal(block(x), fresh(other, cuda_device)(x))
    assert not torch.equal(block(x), before)
    with torch.no_grad():
        block.down.weight.mul_(2)
    assert torch.equal(block(x), fresh(block, cuda_device)(x))
    block.up.weight = torch.nn.Parameter(make(3, cuda_device).up.weight.detach().clone())
    assert torch.equal(block(x), fresh(block, cuda_device)(x))
    block.load_state_dict(make(4, cuda_device).state_dict(), assign=True)
    assert torch.equal(block(x), fresh(block, cuda_device)(x))


def test_weights_are_laid_out_once(cuda_device):
    x = tokens(cuda_device)
    block = make(1, cuda_device).quantize_()
    block(x)
    where = [t.data_ptr() for t in block._fp8]
    block(x)
    assert [t.data_ptr() for t in block._fp8] == where


def test_moves_and_copies_stay_in_8_bits(cuda_device):
    x = tokens(cuda_device)
    block = make(1, cuda_device)
    plain = block(x).detach()
    served = block.quantize_()(x)
    assert not torch.equal(served, plain)
    assert torch.equal(block.to(cuda_device)(x), served)
    assert torch.equal(block.cpu().to(cuda_device)(x), served)
    assert torch.equal(copy.deepcopy(block)(x), served)
    assert torch.equal(block.eval()(x), served)
    assert torch.equal(block.train()(x), plain)


def test_a_block_made_in_inference_mode(cuda_device):
    with torch.inference_mode():
        block = make(1, cuda_device).quantize_()
        out = block(tokens(cuda_device))
    assert torch.equal(out, make(1, cuda_device).quantize_()(tokens(cuda_device)))


def test_inputs_that_want_a_gradient_are_refused(cuda_device):
    x = tokens(cuda_device)
    block = make(1, cuda_device).quantize_()
    want = block(x, x)
    for args in ((x.clone().requires_grad_(), x), (x, x.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            block(*args)
        with torch.no_grad():
            assert torch.equal(block(*args), want)
