"""The serving form reads what the quantisation ahead of it has just written, wherever the
allocator puts that."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,k,n", [(1, 4096, 1024), (1, 1000, 300), (7, 2048, 512),
                                        (40, 640, 4096)], ids=str)
def test_tokens_of_ever_other_sizes_through_one_workspace(tokens, k, n, cuda_device):
    """Rows whose blocks differ by powers of two, call after call: a scale left from the call
    before would be off by a factor of two or more."""
    from sr_states import block_linear, matmul_blocks, quantize_blocks

    gen = torch.Generator().manual_seed(tokens + k)
    w = torch.randn(n, k, generator=gen).to(cuda_device)
    kept = quantize_blocks(w, block=(128, 128))
    blocks = -(-k // 128)
    inputs = []
    for _ in range(100):
        size = torch.randint(-20, 20, (tokens, blocks), generator=gen)
        spread = torch.exp2(size.float()).repeat_interleave(128, 1)[:, :k]
        inputs.append((torch.randn(tokens, k, generator=gen) * spread).to(cuda_device))
    with torch.no_grad():
        # one call behind the other, with nothing between them that waits
        got = [block_linear(x, kept) for x in inputs for _ in range(3)]
        for i, x in enumerate(inputs):
            want = matmul_blocks(quantize_blocks(x), kept, dtype=torch.float32)
            for y in got[3 * i:3 * i + 3]:
                assert torch.equal(y, want), i
