"""The largest numbers of rows that the operators on rows in groups take."""

import pytest
import torch

from sr_states import adapter_linear, expert_linear, group_rows, quantize_blocks
from sr_states.cuda import _native

MOST = 4194240


def test_one_more_is_refused_before_anything_runs():
    from test_host_groups import A, adapters, blocks, refused

    lib = _native.load_library()
    for tokens in (MOST + 1, 2**22):
        refused(lib.srs_adapter_linear(A, tokens, 128, 128, 3, 0, 0, blocks(), adapters(), 0,
                                       A, None, None, A, 1 << 62, None), "out of range")
        turned = dict(square=0, pitch=lib.srs_group_columns(tokens, 2),
                      scale_pitch=lib.srs_group_scales(tokens, 2))
        refused(lib.srs_expert_gradient(blocks(**turned), blocks(**turned), tokens, 2, A, A, 1,
                                        None), "rows must be in")
        refused(lib.srs_expert_linear(A, 1, tokens, 128, 128, 3, blocks(), 2, A, A, A, 1 << 62,
                                      None), "too large")


@pytest.mark.gpu
def test_the_most_rows(cuda_device):
    def make(*shape):
        return torch.randn(shape, device=cuda_device).to(torch.bfloat16)

    x, w, down, up, experts = (make(MOST, 8), make(16, 8), make(3, 2, 8), make(3, 16, 2),
                               make(3, 16, 8))
    index = torch.arange(MOST, device=cuda_device) % 4 - 1
    plan = group_rows(index, 3)
    held = quantize_blocks(w, block=(128, 128))
    picked = torch.tensor([0, 1, 2, 3, MOST // 2, MOST - 4, MOST - 3, MOST - 2, MOST - 1],
                          device=cuda_device)
    y = adapter_linear(x, held, down, up, plan)[picked].double()
    sorted_y = expert_linear(x, experts, plan.ends)
    for place, i in enumerate(picked.tolist()):
        a = (i % 4) - 1
        token = quantize_blocks(x[i:i + 1]).dequantize().double()[0]
        exact = held.dequantize().double() @ token
        sizes = held.dequantize().double().abs() @ token.abs()
        if a >= 0:
            low = down[a].double() @ x[i].double()
            exact = exact + up[a].double() @ low
            sizes = sizes + up[a].double().abs() @ (down[a].double().abs() @ x[i].double().abs())
        # sums of 8 and 2 terms, pairs of BF16, half a step of the result
        limit = 2.0**-16 * sizes + 2.0**-8 * exact.abs()
        assert ((y[place] - exact).abs() <= limit).all()
    ends = plan.ends.tolist()
    for row in (0, ends[0] - 1, ends[0], ends[1] - 1, ends[1], ends[2] - 1):
        e = next(i for i in range(3) if row < ends[i])
        token = quantize_blocks(x[row:row + 1]).dequantize().double()[0]
        matrix = quantize_blocks(experts[e], block=(128, 128)).dequantize().double()
        exact, sizes = matrix @ token, matrix.abs() @ token.abs()
        assert ((sorted_y[row].double() - exact).abs() <=
                2.0**-18 * sizes + 2.0**-8 * exact.abs()).all()
    assert not sorted_y[ends[2]:].any()
    with pytest.raises(ValueError, match="out of range"):
        more = group_rows(torch.zeros(MOST + 1, dtype=torch.int32, device=cuda_device), 3)
        adapter_linear(torch.cat([x, x[:1]]), held, down, up, more)
