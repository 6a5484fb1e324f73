"""Workspaces of the adapters' gradients: as large as what is left in them."""

import pytest
import torch

from sr_states import adapter_linear, group_rows, quantize_blocks
from sr_states.cuda import _native


def test_parts_hold_every_grouping():
    """Few columns, so chunks of 256 tokens: an adapter of up to 256 leaves no part, a larger one a
    part a chunk."""
    call = _native.load_library().srs_adapter_gradient_workspace
    cols, rank = 128, 8
    for tokens in (1, 256, 257, 511, 512, 514, 771, 1000, 5000, 20001):
        size = call(tokens, cols, 50, rank)
        assert size % (4 * cols * rank) == 0
        for each in (257, 300, 512, 513, 600, 769, tokens):
            groups = [each] * (tokens // each) + [tokens % each]
            parts = sum(-(-n // 256) for n in groups if n > 256)
            assert parts * 4 * cols * rank <= size, (tokens, each)
        assert size == call(tokens, cols, 1, rank) == call(tokens, cols, 1024, rank)
    assert call(256, cols, 50, rank) == 0
    assert call(500, 4096 + 14336, 64, 64) < 10 * 2**20
    assert call(0, cols, 50, rank) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,adapters,rank", [(500, 64, 64), (200, 40, 256), (1500, 100, 16)])
def test_gradients_hold_little_beside_their_results(tokens, adapters, rank, cuda_device):
    def make(*shape):
        return torch.randn(shape, device=cuda_device).to(torch.bfloat16)

    x, down, up = make(tokens, 1024), make(adapters, rank, 1024), make(adapters, 2048, rank)
    w = quantize_blocks(make(2048, 1024), block=(128, 128))
    groups = group_rows(torch.arange(tokens, device=cuda_device) % adapters, adapters)
    y = adapter_linear(x, w, down.requires_grad_(), up.requires_grad_(), groups)
    dy = make(*y.shape)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(y, (down, up), dy)
    torch.cuda.synchronize()
    beside = torch.cuda.max_memory_allocated() - before - sum(2 * g.numel() for g in grads)
    # low parts, tokens in blocks and pairs aside: at most 2 parts for every 256 tokens
    assert beside <= 8 * (tokens // 256) * rank * (1024 + 2048) + 40 * tokens * rank + 2**21


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_long_and_short_adapters_side_by_side(dtype, cuda_device):
    """Adapters with and without parts in any order, against FP64."""
    from test_gpu_adapters import run_case

    counts = [300, 20, 700, 1, 0, 513, 256, 257, 0, 40, 900]
    index = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    index = torch.cat([index, torch.full((13,), -1)])
    index = index[torch.randperm(len(index), generator=torch.Generator().manual_seed(1))]
    run_case(len(index), len(counts), 12, 200, 136, dtype, cuda_device, index.to(cuda_device))
