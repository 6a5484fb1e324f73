"""Forward-mode differentiation: the layers on FP8 blocks have no rule for it, and say so."""

import pytest
import torch
import torch.autograd.forward_ad as forward

from sr_states import (BlockTensor, adapter_linear, block_linear, expert_linear, group_rows,
                       quantize_blocks, quantize_stack)
from sr_states.cuda import _native


def dual(t):
    return forward.make_dual(t, torch.ones_like(t))


def test_front_ends_refuse_tangents():
    """Before any CUDA call."""
    x, w = torch.ones((4, 32)), torch.ones((16, 32))
    experts, ends = torch.ones((2, 16, 32)), torch.tensor([2, 4], dtype=torch.int32)
    down, up, order = torch.ones((2, 4, 32)), torch.ones((2, 16, 4)), torch.arange(4).int()
    scale = torch.ones(2)
    held = BlockTensor(w.to(torch.float8_e4m3fn),
                       torch.ones((1, 1)).to(torch.float8_e8m0fnu))
    groups, blocks = _native.groups_module(), _native.blocks_module()

    def adapters(x, w, down, up, scale):
        return groups.adapter_linear(x, w, *(None,) * 4, down, up, scale, 1.0, order, ends, 3, 3, 0,
                                     0)

    with forward.dual_level():
        for call in (lambda: blocks.linear(dual(x), *held, 3),
                     lambda: groups.expert_linear(dual(x), experts, None, ends, 3, 3, 0, 0),
                     lambda: groups.expert_linear(x, dual(experts), None, ends, 3, 3, 0, 0),
                     lambda: adapters(dual(x), w, down, up, scale),
                     lambda: adapters(x, dual(w), down, up, scale),
                     lambda: adapters(x, w, dual(down), up, scale),
                     lambda: adapters(x, w, down, dual(up), scale),
                     lambda: adapters(x, w, down, up, dual(scale))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_layers_refuse_tangents(grad, cuda_device):
    def make(*shape):
        return torch.ones(shape, device=cuda_device, dtype=torch.bfloat16)

    x, w, experts, down, up = (make(4, 32), make(16, 32), make(2, 16, 32), make(2, 4, 32),
                               make(2, 16, 4))
    plan = group_rows(torch.zeros(4, dtype=torch.int32, device=cuda_device), 2)
    held, stack = (quantize_blocks(w, block=(128, 128)), quantize_stack(experts, block=(128, 128)))
    with forward.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda: block_linear(dual(x), w), lambda: block_linear(dual(x), held),
                     lambda: expert_linear(dual(x), experts, plan.ends),
                     lambda: expert_linear(dual(x), stack, plan.ends),
                     lambda: adapter_linear(dual(x), held, down, up, plan),
                     lambda: adapter_linear(x, held, dual(down), up, plan)):
            with pytest.raises(NotImplementedError):
                call()
        # with forward mode switched off, as if there were no tangent
        tangent = dual(x)
        with forward._set_fwd_grad_enabled(False):
            y = adapter_linear(tangent, held, down, up, plan)
            assert torch.equal(y, adapter_linear(x, held, down, up, plan))
            assert torch.equal(expert_linear(tangent, stack, plan.ends),
                               expert_linear(x, stack, plan.ends))
