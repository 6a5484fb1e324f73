"""Results that are changed in place, as a residual added to a layer's result is."""

import pytest
import torch

from sr_states import adapter_linear, block_linear, expert_linear, group_rows, quantize_blocks

pytestmark = pytest.mark.gpu

SHAPES = pytest.mark.parametrize("shape", [(64,), (6, 64), (2, 3, 64), (2, 1, 3, 64), (0, 3, 64)],
                                 ids=lambda s: "x".join(map(str, s)))


def values(shape, seed, device):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(device, torch.bfloat16)


def check(call, x, leaves):
    """y += residual gives what y + residual gives, and the residual gets its gradient."""
    residual = values((*x.shape[:-1], 48), 7, x.device).requires_grad_()
    dy = values(residual.shape, 8, x.device)
    y = call() + residual
    want = torch.autograd.grad(y, (residual, *leaves), dy)
    got = call()
    got += residual
    got.mul_(1)
    assert torch.equal(got, y)
    for a, b in zip(torch.autograd.grad(got, (residual, *leaves), dy), want):
        assert a.shape == b.shape and torch.equal(a, b)


@SHAPES
@pytest.mark.parametrize("frozen", [True, False])
def test_adapters(shape, frozen, cuda_device):
    x = values(shape, 1, cuda_device).requires_grad_()
    w = values((48, 64), 2, cuda_device)
    down = values((2, 8, 64), 3, cuda_device).requires_grad_()
    up = values((2, 48, 8), 4, cuda_device).requires_grad_()
    tokens = x.numel() // 64
    plan = group_rows(torch.arange(tokens, device=cuda_device) % 3, 2)
    if frozen:
        held = quantize_blocks(w, block=(128, 128), orientation="both")
        check(lambda: adapter_linear(x, held, down, up, plan, seed=3), x, (x, down, up))
    else:
        w.requires_grad_()
        check(lambda: adapter_linear(x, w, down, up, plan, seed=3), x, (x, w, down, up))


def test_experts(cuda_device):
    x = values((6, 64), 1, cuda_device).requires_grad_()
    w = values((2, 48, 64), 2, cuda_device).requires_grad_()
    ends = torch.tensor([2, 5], device=cuda_device)
    check(lambda: expert_linear(x, w, ends, seed=3), x, (x, w))


@SHAPES
def test_one_weight(shape, cuda_device):
    x = values(shape, 1, cuda_device).requires_grad_()
    w = values((48, 64), 2, cuda_device).requires_grad_()
    check(lambda: block_linear(x, w, seed=3), x, (x, w))
