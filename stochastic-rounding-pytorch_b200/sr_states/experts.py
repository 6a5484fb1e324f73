"""Linear layers of a mixture of experts: rows in groups, one weight a group, products in FP8
blocks (forward and both gradients).

Rounding is ``block_linear``'s.  The blocks of 128 rows that a weight's gradient sums over are
counted from its expert's first row, so an expert's gradient does not depend on what the others
hold.
"""

from __future__ import annotations

import torch

from .blocks import BlockLayer
from .cuda.blocks import BLOCK, BlockTensor, check_blocks, quantize_blocks, quantize_stack
from .cuda.groups import expert_blocks, expert_gradient, expert_matmul, quantize_groups

__all__ = ["BlockExperts", "expert_linear"]


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends, dtype, grad_dtype, grad_rounding, seed, need_x, need_w):
        tokens_t = matrix_t = None
        if need_w:
            tokens, tokens_t = quantize_groups(x, ends, dtype=dtype, rows=True)
        else:
            tokens = quantize_blocks(x, dtype=dtype)
        matrix = quantize_stack(weight, dtype=dtype, block=(BLOCK, BLOCK),
                                orientation="both" if need_x else "rows")
        matrix, matrix_t = matrix if need_x else (matrix, None)
        ctx.save_for_backward(ends, *(tokens_t or ()), *(matrix_t or ()))
        ctx.settings = (grad_dtype, grad_rounding, seed, x.dtype, weight.dtype, need_x, need_w)
        return expert_matmul(tokens, matrix, ends, dtype=x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        grad_dtype, rounding, seed, x_dtype, w_dtype, need_x, need_w = ctx.settings
        ends, *saved = ctx.saved_tensors
        tokens_t = BlockTensor(saved.pop(0), saved.pop(0)) if need_w else None
        matrix_t = BlockTensor(saved.pop(0), saved.pop(0)) if need_x else None
        how = {"dtype": grad_dtype, "rounding": rounding, "seed": seed}
        rows = columns = None
        if need_w:
            got = quantize_groups(dy, ends, rows=need_x, **how)
            rows, columns = got if need_x else (None, got)
        elif need_x:
            rows = quantize_blocks(dy, **how)
        dx = expert_matmul(rows, matrix_t, ends, dtype=x_dtype) if need_x else None
        dw = (expert_gradient(columns, tokens_t, dy.shape[0], ends, dtype=w_dtype)
              if need_w else None)
        return dx, dw, None, None, None, None, None, None, None


def expert_linear(x, weight, ends, *, dtype=torch.float8_e4m3fn, grad_dtype=torch.float8_e4m3fn,
                  grad_rounding="stochastic", seed=0):
    """``x[i] @ weight[e].T`` for the rows ``ends[e - 1] <= i < ends[e]`` of expert e, with FP8
    block products; rows from ``ends[-1]`` on belong to no expert and give zeros.

    ``x``: (rows, K) in FP32, BF16 or FP16, sorted by expert; ``ends``: int32 or int64 on the
    same GPU, one entry an expert (at most 1024), rising, as ``group_rows`` gives them (the host
    does not read it).  ``weight``: an (experts, N, K) tensor (quantised in the call;
    differentiable in ``x`` and ``weight``), or a BlockTensor kept from ``quantize_stack``
    (inference).  The rest as for ``block_linear``.  At most 2^22 rows and 2^30 rows of weights.
    """
    stack = (weight.data if isinstance(weight, BlockTensor) else weight).shape
    if x.dim() != 2 or len(stack) != 3 or x.shape[1] != stack[2]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit expert weights of shape "
                         f"{tuple(stack)}")
    if ends.dim() != 1 or ends.shape[0] != stack[0]:
        raise ValueError(f"ends of shape {tuple(ends.shape)} do not fit {stack[0]} experts")
    if isinstance(weight, BlockTensor):
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("a BlockTensor weight has no backward pass; pass the weight itself "
                             "or run under torch.no_grad()")
        return expert_blocks(x, weight, ends, dtype)
    check_blocks(grad_dtype, grad_rounding)
    grad = torch.is_grad_enabled()
    return _ExpertLinear.apply(x, weight, ends, dtype, grad_dtype, grad_rounding, seed,
                               grad and x.requires_grad, grad and weight.requires_grad)


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
