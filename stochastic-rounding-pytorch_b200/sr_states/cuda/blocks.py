"""FP8 blocks on the sm_100a kernels: quantisation and block-scaled products."""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..rounding import native_codes
from . import _native

BLOCK = 128
ORIENTATIONS = {"rows": 1, "columns": 2, "both": 3}
_MASK32 = 0xFFFFFFFF
_FORMATS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FP8 = {torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}


class BlockTensor(NamedTuple):
    """A matrix in FP8 blocks: element (i, j) stands for data[i, j] * scale of its block.

    ``data``: E4M3 or E5M2, rows x columns; ``scale``: float8_e8m0fnu (powers of
    two), one a 1 x 128 block (rows x ceil(columns / 128)) or one a 128 x 128 block
    (ceil(rows / 128) x ceil(columns / 128))."""

    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The values the blocks stand for."""
        rows, cols = self.data.shape
        factor = self.scale.float().repeat_interleave(BLOCK, 1)[:, :cols]
        if self.scale.shape[0] != rows:
            factor = factor.repeat_interleave(BLOCK, 0)[:rows]
        return (self.data.float() * factor).to(dtype)


def check_blocks(dtype, rounding):
    """The entry points' codes of a block format and a rounding rule."""
    if dtype not in _FP8:
        raise TypeError(f"blocks are held in float8_e4m3fn or float8_e5m2, got {dtype}")
    return native_codes(dtype, rounding)


def quantize_blocks(x, *, dtype=torch.float8_e4m3fn, rounding="nearest", seed=0, offset=0,
                    block=(1, BLOCK), orientation="rows"):
    """Quantise a matrix to FP8 blocks of 128, read once.

    Per block: k is the smallest exponent (at least -127) with
    max|x| <= largest * 2^k over its finite elements (0 if all are zero), the scale is
    2^k and the data are x * 2^-k rounded by ``rounding``; infinities saturate, NaN
    is kept.  ``block``: ``(1, 128)`` or ``(128, 128)``.

    ``orientation``: ``"rows"`` gives the BlockTensor of ``x`` (blocks along its
    rows), ``"columns"`` that of its transpose (blocks along its columns), ``"both"``
    the pair.  Stochastic counters: element (i, j) of ``x`` uses the hash of its
    flat index + offset + state_key(seed, 0), its transposed copy state_key(seed, 1).

    ``x``: FP32, BF16 or FP16 on an sm_100a GPU, two dimensions, at most 4194240 rows.
    """
    fmt, rule = check_blocks(dtype, rounding)
    if tuple(block) not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, {BLOCK}) or ({BLOCK}, {BLOCK})")
    if orientation not in ORIENTATIONS:
        raise ValueError(f"orientation must be one of {tuple(ORIENTATIONS)}")
    launcher = _native.launcher()
    launcher.check_device(x.device, "quantize_blocks")
    got = launcher.quantize_blocks(x, fmt, rule, int(block[0] == BLOCK), int(seed) & _MASK32,
                                   int(offset) & _MASK32, ORIENTATIONS[orientation])
    if orientation == "both":
        return BlockTensor(got[0], got[1]), BlockTensor(got[2], got[3])
    return BlockTensor(*got)


def matmul_blocks(a, b, *, dtype=torch.bfloat16):
    """``a @ b.T`` of two BlockTensors (a: M x K, b: N x K), summed in FP32.

    Either operand may be E4M3 or E5M2 with scales of either block form; the
    result is FP32, BF16 or FP16.  The tensor core truncates the terms of its sums: an
    element is within (K + 2) 2^-23 of the sum of its terms' sizes.  K = 0 gives zeros; K is
    at most 2^30.  Data whose rows do not start on 16-byte boundaries are copied once (those
    of ``quantize_blocks`` do)."""
    if dtype not in _FORMATS:
        raise TypeError(f"matmul_blocks gives FP32, BF16 or FP16, got {dtype}")
    launcher = _native.launcher()
    (a_data, a_scale), (b_data, b_scale) = a, b
    launcher.check_device(a_data.device, "matmul_blocks")
    return launcher.matmul_blocks(a_data, a_scale, b_data, b_scale, _FORMATS[dtype])


def linear_blocks(x, weight, dtype):
    """``x @ weight.T`` of a tensor quantised to nearest in rows and a BlockTensor kept
    by the caller, in one call; the result has x's dtype."""
    launcher = _native.launcher()
    launcher.check_device(x.device, "block_linear")
    if dtype not in _FP8:
        raise TypeError(f"blocks are held in float8_e4m3fn or float8_e5m2, got {dtype}")
    return launcher.block_linear(x, weight.data, weight.scale, _FP8[dtype])
