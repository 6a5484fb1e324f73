"""The longest sums that a product takes: seconds in one tile, and no wait gives up."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_product_of_the_longest_rows(cuda_device):
    """65 rows (one more than the thin form takes) of 2^30 elements, 70 GB; small integers in a
    few places, so that the sums are exact."""
    from sr_states import BlockTensor, matmul_blocks
    from sr_states.cuda import check_products

    rows, k = 65, 1 << 30
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of free memory")
    data = torch.zeros((rows, k), dtype=torch.uint8, device=cuda_device)
    scale = torch.full((rows, k // 128), 127, dtype=torch.uint8, device=cuda_device)
    values = torch.zeros((rows, 64), device=cuda_device)
    gen = torch.Generator().manual_seed(1)
    for at, part in zip((0, 1 << 20, k // 2 + 77, k - 16), range(4)):
        some = torch.randint(-4, 5, (rows, 16), generator=gen).float().to(cuda_device)
        data[:, at:at + 16] = some.to(torch.float8_e4m3fn).view(torch.uint8)
        values[:, 16 * part:16 * part + 16] = some
    a = BlockTensor(data.view(torch.float8_e4m3fn), scale.view(torch.float8_e8m0fnu))
    d = matmul_blocks(a, a, dtype=torch.float32)
    check_products(cuda_device)
    assert torch.equal(d, values @ values.T)
    del a, data, scale
    torch.cuda.empty_cache()
