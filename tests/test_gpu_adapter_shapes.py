"""Adapters at sizes where the products of few tokens change their tiles, and the digits of FP16
low parts of tokens of very different sizes."""

import pytest
import torch

from sr_states import adapter_linear, group_rows, quantize_blocks
from test_gpu_adapters import HALF_ULP, U, indices, run_case, values


def pairs(h, top):
    """FP64 numbers as the pairs of FP16 that hold them, scaled so that `top` is 2^13 .. 2^14."""
    factor = 2.0 ** (13 - torch.floor(torch.log2(top)).clamp(-17, 73))
    high = (h * factor).half()
    rest = (h * factor - high.double()).half()
    return (high.double() + rest.double()) / factor


def lost(h, top):
    """What such a pair loses: high and rest have 11 bits each, and below 2^-14 steps of 2^-24."""
    return 2.0**-22 * h.abs() + 2.0**-38 * top + 2.0**-55


def test_the_bound_tells_a_tokens_own_scale_from_the_batchs():
    gen = torch.Generator().manual_seed(1)
    h = torch.randn((64, 16), generator=gen, dtype=torch.float64)
    h *= 2.0 ** torch.linspace(-14, 12, 64)[:, None]
    own = h.abs().amax(1, keepdim=True)
    assert ((pairs(h, own) - h).abs() <= lost(h, own)).all()
    assert not ((pairs(h, h.abs().max()) - h).abs() <= lost(h, own)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 20, 100])
@pytest.mark.parametrize("tokens", [40, 64, 300])
def test_small_tokens_beside_large_ones_of_their_adapter(tokens, rank, cuda_device):
    """No projection beside the adapters' part, so that the small tokens' digits show."""
    k, n = 96, 72
    size = 2.0 ** (torch.arange(tokens) * 11 % 27 - 14).to(cuda_device)
    x = (values((tokens, k), 1, cuda_device, torch.float32) * size[:, None]).half()
    down = values((2, rank, k), 2, cuda_device, torch.float16, 0.3 * k**-0.5)
    up = values((2, n, rank), 3, cuda_device, torch.float16, 0.3 * rank**-0.5)
    w = quantize_blocks(torch.zeros((n, k), device=cuda_device, dtype=torch.float16),
                        block=(128, 128))
    index = torch.arange(tokens, device=cuda_device) % 3 - 1
    with torch.no_grad():
        y = adapter_linear(x, w, down, up, group_rows(index, 2)).double()
    assert not y[index == -1].any()
    for a in range(2):
        rows = index == a
        t, d, u = x[rows].double(), down[a].double(), up[a].double()
        h = t @ d.mT
        off = (k + 16) * U * (t.abs() @ d.abs().mT) + lost(h, h.abs().amax(1, keepdim=True))
        exact = h @ u.mT
        error = off @ u.abs().mT + (2 * rank + 8) * U * (h.abs() @ u.abs().mT)
        limit = error + HALF_ULP[torch.float16] * (exact.abs() + error) + 2.0**-25
        assert ((y[rows] - exact).abs() <= limit).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,adapters", [(1, 1), (20, 30), (64, 90)])
@pytest.mark.parametrize("rank", [8, 20, 64])
@pytest.mark.parametrize("k,n", [(130, 19000), (96, 28672), (19000, 130), (1, 1), (8, 18945)])
def test_few_tokens_by_matrices_of_more_tiles_than_sms(tokens, adapters, rank, k, n, cuda_device):
    """Tiles of fewer than 128 rows forward, whole ones backward, k not split."""
    dtype = torch.bfloat16 if rank == 20 else torch.float16
    run_case(tokens, adapters, rank, k, n, dtype, cuda_device,
             indices(tokens, adapters, "mixed", cuda_device, seed=tokens))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [30, 200])
def test_one_matrix_for_all_adapters(tokens, cuda_device):
    """Stacks that are views of one matrix: values as of copies, and a gradient for the matrix."""
    down = values((8, 128), 1, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    up = values((96, 8), 2, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    x = values((tokens, 128), 3, cuda_device, torch.bfloat16).requires_grad_()
    w = quantize_blocks(values((96, 128), 4, cuda_device, torch.bfloat16), block=(128, 128),
                        orientation="both")
    dy = values((1, 96), 5, cuda_device, torch.bfloat16).expand(tokens, 96)  # broadcast, too
    plan = group_rows(torch.arange(tokens, device=cuda_device) % 4 - 1, 3)

    def run(spread):
        y = adapter_linear(x, w, spread(down), spread(up), plan, seed=2)
        return (y, *torch.autograd.grad(y, (x, down, up), dy))

    views = run(lambda m: m.expand(3, *m.shape))
    copies = run(lambda m: torch.stack([m] * 3))
    for a, b in zip(views[:2], copies[:2]):
        assert torch.equal(a, b)
    for a, b in zip(views[2:], copies[2:]):
        # sums of three BF16 numbers, in two orders
        assert ((a.double() - b.double()).abs() <= 2.0**-7 * b.double().abs() +
                2.0**-7 * b.double().abs().amax()).all()
