"""Low-rank adapters of many requests at once beside a projection in FP8 blocks.

The projection is ``block_linear``'s; the adapters' part is computed from the tokens and matrices
as they are (FP32 sums), and the sum of both is rounded once.
"""

from __future__ import annotations

import torch

from .cuda import _native
from .cuda.blocks import BlockTensor, check_blocks

__all__ = ["adapter_linear"]


def adapter_linear(x, weight, down, up, groups, *, scale=1.0, dtype=torch.float8_e4m3fn,
                   grad_dtype=torch.float8_e4m3fn, grad_rounding="stochastic", seed=0):
    """``block_linear(x, weight)`` plus, for the tokens t of adapter a,
    ``scale[a] * (x[t] @ down[a].T) @ up[a].T``, rounded once.

    ``x``: (..., K) in BF16 or FP16; ``down``: (adapters, rank, K) and ``up``: (adapters, N,
    rank) in x's dtype, rank at most 256; ``groups``: the tokens (x's rows taken flat) by adapter, from
    ``group_rows(index, adapters)``: made once a batch, for all its layers.  Tokens of no group
    have the projection alone.  Infinities and NaN in an adapter's matrices reach its own tokens
    alone (as either).  ``scale``: a number, or FP32, one an adapter (no gradient).

    ``weight``: a BlockTensor (inference), a pair of BlockTensors
    ``quantize_blocks(w, block=(128, 128), orientation="both")`` (a frozen projection:
    differentiable in ``x``, ``down`` and ``up``), or an (N, K) tensor (quantised in the call,
    differentiable too).  The rest as for ``block_linear``.  At most 4194240 tokens.
    """
    kept = turned = (None, None)
    if isinstance(weight, BlockTensor):
        kept, weight = weight, None
    elif isinstance(weight, (tuple, list)):
        if len(weight) != 2 or not all(isinstance(w, BlockTensor) for w in weight):
            raise TypeError("a kept weight is a BlockTensor or a pair of them")
        (kept, turned), weight = weight, None
    fmt, _ = check_blocks(dtype, "nearest")
    grad_fmt, grad_rule = check_blocks(grad_dtype, grad_rounding)
    launcher = _native.launcher()
    launcher.check_device(x.device, "adapter_linear")
    scale, factor = (scale, 1.0) if isinstance(scale, torch.Tensor) else (None, float(scale))
    return launcher.adapter_linear(x, weight, kept, turned, down, up, scale, factor, groups.order,
                                   groups.ends, fmt, grad_fmt, grad_rule, int(seed) & 0xFFFFFFFF)
