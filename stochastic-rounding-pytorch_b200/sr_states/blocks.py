"""Linear layers whose products run in FP8 blocks (forward and both gradients).

Weights and activations are rounded to nearest; gradients stochastically, so
that the weight gradient's expectation is the exact product's and small gradients
are not lost.  Blocks are 1 x 128 along the summed dimension for activations and
gradients and 128 x 128 for weights.
"""

from __future__ import annotations

import itertools

import torch

from ._hash import update_key
from .cuda.blocks import (BLOCK, BlockTensor, check_blocks, linear_blocks, matmul_blocks,
                          quantize_blocks, quantize_stack)

__all__ = ["BlockLinear", "BlockTensor", "block_linear", "matmul_blocks", "quantize_blocks",
           "quantize_stack"]


def _matrix(x):
    # all but the last dimension in one; sizes of zero included, unlike reshape(-1, K)
    return x if x.dim() == 2 else x.flatten(0, -2) if x.dim() > 1 else x.unsqueeze(0)


class _BlockLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, dtype, grad_dtype, grad_rounding, seed, need_x, need_w):
        tokens = quantize_blocks(_matrix(x), dtype=dtype,
                                 orientation="both" if need_w else "rows")
        matrix = quantize_blocks(weight, dtype=dtype, block=(BLOCK, BLOCK),
                                 orientation="both" if need_x else "rows")
        tokens, tokens_t = tokens if need_w else (tokens, None)
        matrix, matrix_t = matrix if need_x else (matrix, None)
        ctx.save_for_backward(*(tokens_t or ()), *(matrix_t or ()))
        ctx.settings = (grad_dtype, grad_rounding, seed, x.shape, x.dtype, weight.dtype, need_x,
                        need_w)
        y = matmul_blocks(tokens, matrix, dtype=x.dtype)
        if x.dim() == 2:
            return y
        # no view: autograd refuses to change one in place that was made inside a function
        return torch.ops.aten._unsafe_view(y, (*x.shape[:-1], weight.shape[0]))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        grad_dtype, rounding, seed, shape, x_dtype, w_dtype, need_x, need_w = ctx.settings
        saved = list(ctx.saved_tensors)
        tokens_t = BlockTensor(saved.pop(0), saved.pop(0)) if need_w else None
        matrix_t = BlockTensor(saved.pop(0), saved.pop(0)) if need_x else None
        orientation = "both" if need_x and need_w else "rows" if need_x else "columns"
        got = quantize_blocks(_matrix(dy), dtype=grad_dtype, rounding=rounding, seed=seed,
                              orientation=orientation)
        rows, columns = got if orientation == "both" else (got, got)
        dx = matmul_blocks(rows, matrix_t, dtype=x_dtype).reshape(shape) if need_x else None
        dw = matmul_blocks(columns, tokens_t, dtype=w_dtype) if need_w else None
        return dx, dw, None, None, None, None, None, None


def block_linear(x, weight, *, dtype=torch.float8_e4m3fn, grad_dtype=torch.float8_e4m3fn,
                 grad_rounding="stochastic", seed=0):
    """``x @ weight.T`` with FP8 block products; ``x``: (..., K) in FP32, BF16 or FP16.

    ``weight``: an (N, K) tensor (quantised in the call; differentiable in ``x`` and
    ``weight``), or a BlockTensor kept from ``quantize_blocks`` (inference).
    ``grad_dtype`` and ``grad_rounding`` are those of the output gradient in the
    backward products; ``seed`` is its rounding's seed (a new one every step).
    """
    if x.dim() < 1:
        raise ValueError("block_linear needs at least one dimension")
    columns = (weight.data if isinstance(weight, BlockTensor) else weight).shape
    if len(columns) != 2 or x.shape[-1] != columns[1]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit a weight of shape "
                         f"{tuple(columns)}")
    if isinstance(weight, BlockTensor):
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("a BlockTensor weight has no backward pass; pass the weight itself "
                             "or run under torch.no_grad()")
        return linear_blocks(x, weight, dtype)
    check_blocks(grad_dtype, grad_rounding)
    # asked here: inside a Function inputs "need" gradients under torch.no_grad() as well
    grad = torch.is_grad_enabled()
    return _BlockLinear.apply(x, weight, dtype, grad_dtype, grad_rounding, seed,
                              grad and x.requires_grad, grad and weight.requires_grad)


def _rank():
    distributed = torch.distributed
    if distributed.is_available() and distributed.is_initialized():
        return distributed.get_rank()
    return 0


class BlockLayer(torch.nn.Module):
    """The weight of a layer on FP8 block products, and the draws of its gradient's rounding."""

    _made = itertools.count()

    def __init__(self, *shape, grad_dtype=torch.float8_e4m3fn, grad_rounding="stochastic",
                 seed=None, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.out_features, self.in_features = shape[-2:]
        self.grad_dtype, self.grad_rounding = grad_dtype, grad_rounding
        self.seed, self.calls = int(next(self._made) if seed is None else seed), 0
        self.weight = torch.nn.Parameter(torch.empty(shape, device=device, dtype=dtype))
        torch.nn.init.normal_(self.weight, std=self.in_features ** -0.5)

    def get_extra_state(self):
        return torch.tensor([self.seed, self.calls], dtype=torch.int64)

    def set_extra_state(self, state):
        self.seed, self.calls = (int(v) for v in state)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)
        # a state_dict of the weight alone is whole, too
        key = prefix + "_extra_state"
        if key in missing_keys:
            missing_keys.remove(key)

    def quantized(self) -> BlockTensor:
        """The weight in FP8 blocks, to keep for inference."""
        return quantize_blocks(self.weight, block=(BLOCK, BLOCK))

    def _settings(self, x):
        """The gradient's settings for one call on ``x``."""
        if torch.is_grad_enabled() and (x.requires_grad or self.weight.requires_grad):
            self.calls += 1
        return {"grad_dtype": self.grad_dtype, "grad_rounding": self.grad_rounding,
                "seed": update_key(self.seed, self.calls, _rank())}


class BlockLinear(BlockLayer):
    """A linear layer without bias on ``block_linear``.

    The gradient's rounding draws anew on every call that a gradient will follow:
    (seed, number of such calls, rank of the process).  ``seed=None`` gives a layer the
    number of layers that the process made before it, so that layers draw apart.  The
    ``state_dict`` carries the seed and the calls: a run that goes on from a checkpoint
    rounds as the run that wrote it would have.
    """

    def __init__(self, in_features, out_features, *, grad_dtype=torch.float8_e4m3fn,
                 grad_rounding="stochastic", seed=None, device=None, dtype=torch.bfloat16):
        super().__init__(out_features, in_features, grad_dtype=grad_dtype,
                         grad_rounding=grad_rounding, seed=seed, device=device, dtype=dtype)

    def forward(self, x):
        return block_linear(x, self.weight, **self._settings(x))
