"""Linear layers of a mixture of experts: rows in groups, one weight a group, products in FP8
blocks (forward and both gradients).

Rounding is ``block_linear``'s.  The blocks of 128 rows that a weight's gradient sums over are
counted from its expert's first row, so an expert's gradient does not depend on what the others
hold.
"""

from __future__ import annotations

import torch

from .blocks import BlockLayer
from .cuda import _native
from .cuda.blocks import BLOCK, BlockTensor, check_blocks, quantize_stack

__all__ = ["BlockExperts", "expert_linear"]


def expert_linear(x, weight, ends, *, dtype=torch.float8_e4m3fn, grad_dtype=torch.float8_e4m3fn,
                  grad_rounding="stochastic", seed=0):
    """``x[i] @ weight[e].T`` for the rows ``ends[e - 1] <= i < ends[e]`` of expert e, with FP8
    block products; rows from ``ends[-1]`` on belong to no expert and give zeros.

    ``x``: (rows, K) in FP32, BF16 or FP16, sorted by expert; ``ends``: int32 or int64 on the
    same GPU, one entry an expert (at most 1024), rising, as ``group_rows`` gives them (the host
    does not read it).  ``weight``: an (experts, N, K) tensor (quantised in the call;
    differentiable in ``x`` and ``weight``), or a BlockTensor kept from ``quantize_stack``
    (inference).  The rest as for ``block_linear``.  At most 4194240 rows and 2^30 rows of
    weights.
    """
    fmt, _ = check_blocks(dtype, "nearest")
    grad_fmt, grad_rule = check_blocks(grad_dtype, grad_rounding)
    launcher = _native.launcher()
    launcher.check_device(x.device, "expert_linear")
    weight, scale = weight if isinstance(weight, BlockTensor) else (weight, None)
    return launcher.expert_linear(x, weight, scale, ends, fmt, grad_fmt, grad_rule,
                                  int(seed) & 0xFFFFFFFF)


class BlockExperts(BlockLayer):
    """Expert layers without bias on ``expert_linear``, beside ``BlockLinear``: same draws, same
    ``state_dict``."""

    def __init__(self, experts, in_features, out_features, *, grad_dtype=torch.float8_e4m3fn,
                 grad_rounding="stochastic", seed=None, device=None, dtype=torch.bfloat16):
        super().__init__(experts, out_features, in_features, grad_dtype=grad_dtype,
                         grad_rounding=grad_rounding, seed=seed, device=device, dtype=dtype)
        self.experts = experts

    def quantized(self) -> BlockTensor:
        """The weights in FP8 blocks, to keep for inference."""
        return quantize_stack(self.weight, block=(BLOCK, BLOCK))

    def forward(self, x, ends):
        return expert_linear(x, self.weight, ends, **self._settings(x))
