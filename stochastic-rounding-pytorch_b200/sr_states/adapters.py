"""Low-rank adapters of many requests at once beside a projection in FP8 blocks.

The projection is ``block_linear``'s; the adapters' part is computed from the tokens and matrices
as they are (FP32 sums), and the sum of both is rounded once.
"""

from __future__ import annotations

import torch

from .blocks import _matrix
from .cuda.blocks import BLOCK, BlockTensor, check_blocks, matmul_blocks, quantize_blocks
from .cuda.groups import Low, RowGroups, adapter_gradient, adapter_product

__all__ = ["adapter_linear"]


class _AdapterLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, down, up, kept, groups, scale, dtype, grad_dtype, grad_rounding,
                seed, need):
        need_x, need_w, need_down, need_up = need
        flat = _matrix(x)
        if kept is not None:
            matrix, matrix_t = kept
        else:
            got = quantize_blocks(weight, dtype=dtype, block=(BLOCK, BLOCK),
                                  orientation="both" if need_x else "rows")
            matrix, matrix_t = got if need_x else (got, None)
        y, low = adapter_product(flat, matrix, down, up, groups, scale=scale, dtype=dtype,
                                 keep=need_up)
        tokens_t = quantize_blocks(flat, dtype=dtype, orientation="columns") if need_w else None
        parts = {"groups": groups, "down": (down,), "up": (up,), "low": low,
                 "x": (flat,) if need_down else (), "tokens": tokens_t or (),
                 "matrix": matrix_t if need_x else (),
                 "scale": (scale,) if isinstance(scale, torch.Tensor) else ()}
        parts = {name: tuple(t for t in given if t is not None) for name, given in parts.items()}
        ctx.save_for_backward(*(t for given in parts.values() for t in given))
        ctx.sizes = {name: len(given) for name, given in parts.items()}
        ctx.settings = (grad_dtype, grad_rounding, seed, x.shape, x.dtype,
                        None if weight is None else weight.dtype,
                        None if isinstance(scale, torch.Tensor) else scale, need)
        return y.reshape(*x.shape[:-1], up.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        grad_dtype, rounding, seed, shape, x_dtype, w_dtype, scale, need = ctx.settings
        need_x, need_w, need_down, need_up = need
        saved, at = {}, 0
        for name, size in ctx.sizes.items():
            saved[name] = ctx.saved_tensors[at:at + size]
            at += size
        groups, (down,), (up,) = RowGroups(*saved["groups"]), saved["down"], saved["up"]
        scale = saved["scale"][0] if saved["scale"] else scale
        flat = _matrix(dy)
        dx = dw = ddown = dup = None
        if need_x or need_down:
            dx, back = adapter_product(
                flat, BlockTensor(*saved["matrix"]) if need_x else None, down, up, groups,
                scale=scale, dtype=grad_dtype, rounding=rounding, seed=seed, turned=True,
                keep=need_down)
            dx = dx.reshape(shape) if need_x else None
        if need_down:
            ddown = adapter_gradient(saved["x"][0], back, groups)
        if need_up:
            dup = adapter_gradient(flat, _low(saved["low"]), groups, turned=True)
        if need_w:
            columns = quantize_blocks(flat, dtype=grad_dtype, rounding=rounding, seed=seed,
                                      orientation="columns")
            dw = matmul_blocks(columns, BlockTensor(*saved["tokens"]), dtype=w_dtype)
        return dx, dw, ddown, dup, *[None] * 8


def _low(saved):
    return Low(saved[0], saved[1] if len(saved) > 1 else None)


def adapter_linear(x, weight, down, up, groups, *, scale=1.0, dtype=torch.float8_e4m3fn,
                   grad_dtype=torch.float8_e4m3fn, grad_rounding="stochastic", seed=0):
    """``block_linear(x, weight)`` plus, for the tokens t of adapter a,
    ``scale[a] * (x[t] @ down[a].T) @ up[a].T``, rounded once.

    ``x``: (..., K) in BF16 or FP16; ``down``: (adapters, rank, K) and ``up``: (adapters, N,
    rank) in x's dtype, rank at most 256; ``groups``: the tokens (x's rows taken flat) by adapter, from
    ``group_rows(index, adapters)``: made once a batch, for all its layers.  Tokens of no group
    have the projection alone.  ``scale``: a number, or FP32, one an adapter (no gradient).

    ``weight``: a BlockTensor (inference), a pair of BlockTensors
    ``quantize_blocks(w, block=(128, 128), orientation="both")`` (a frozen projection:
    differentiable in ``x``, ``down`` and ``up``), or an (N, K) tensor (quantised in the call,
    differentiable too).  The rest as for ``block_linear``.  At most 2^22 tokens.  With FP16
    the inner products must stay below 65504.
    """
    if x.dim() < 1:
        raise ValueError("adapter_linear needs at least one dimension")
    kept = None
    if isinstance(weight, BlockTensor):
        kept, weight = (weight, None), None
    elif isinstance(weight, (tuple, list)):
        if len(weight) != 2 or not all(isinstance(w, BlockTensor) for w in weight):
            raise TypeError("a kept weight is a BlockTensor or a pair of them")
        kept, weight = tuple(weight), None
        rows, columns = kept[0].data.shape, kept[1].data.shape
        if tuple(rows) != tuple(columns)[::-1]:
            raise ValueError(f"blocks of shapes {tuple(rows)} and {tuple(columns)} are not of a "
                             "matrix and its transpose")
    sizes = (kept[0].data if kept is not None else weight).shape
    if len(sizes) != 2 or x.shape[-1] != sizes[1]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit a weight of shape "
                         f"{tuple(sizes)}")
    check_blocks(grad_dtype, grad_rounding)
    grad = torch.is_grad_enabled()
    need = tuple(grad and t is not None and t.requires_grad for t in (x, weight, down, up))
    if not any(need):
        flat = _matrix(x)
        if kept is None:
            kept = (quantize_blocks(weight, dtype=dtype, block=(BLOCK, BLOCK)), None)
        y, _ = adapter_product(flat, kept[0], down, up, groups, scale=scale, dtype=dtype)
        return y.reshape(*x.shape[:-1], sizes[0])
    if kept is not None and kept[1] is None and need[0]:
        raise ValueError("a BlockTensor weight has no backward pass; pass the blocks of both "
                         "orientations or the weight itself, or run under torch.no_grad()")
    return _AdapterLinear.apply(x, weight, down, up, kept, groups, scale, dtype, grad_dtype,
                                grad_rounding, seed, need)
