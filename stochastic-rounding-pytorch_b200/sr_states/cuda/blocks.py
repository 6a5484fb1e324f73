"""FP8 blocks on the sm_100a kernels: quantisation and block-scaled products."""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..rounding import native_codes
from . import _native
from ._launch import device_guard, stream_handle

BLOCK = 128
ORIENTATIONS = ("rows", "columns", "both")
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


def _empty_blocks(rows, cols, dtype, square, device) -> BlockTensor:
    # Row pitches of 16 bytes' multiples, as the products' copies need them.
    pitch = -(-cols // 16) * 16
    data = torch.empty((rows, pitch), dtype=dtype, device=device)
    scale = torch.empty((-(-rows // BLOCK) if square else rows, -(-cols // BLOCK)),
                        dtype=torch.float8_e8m0fnu, device=device)
    return BlockTensor(data if pitch == cols else data[:, :cols], scale)


def _addresses(t):
    if t is None:
        return None, 0, None, 0
    return t.data.data_ptr(), t.data.stride(0), t.scale.data_ptr(), t.scale.stride(0)


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

    ``x``: FP32, BF16 or FP16 on an sm_100a GPU, two dimensions.
    """
    if dtype not in _FP8:
        raise TypeError(f"blocks are held in float8_e4m3fn or float8_e5m2, got {dtype}")
    fmt, rule = native_codes(dtype, rounding)
    if tuple(block) not in ((1, BLOCK), (BLOCK, BLOCK)):
        raise ValueError(f"block must be (1, {BLOCK}) or ({BLOCK}, {BLOCK})")
    if orientation not in ORIENTATIONS:
        raise ValueError(f"orientation must be one of {ORIENTATIONS}")
    launcher = _native.launcher()
    launcher.check_device(x.device, "quantize_blocks")
    if x.dtype not in _FORMATS:
        raise TypeError(f"quantize_blocks takes FP32, BF16 or FP16, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"quantize_blocks needs a matrix, got shape {tuple(x.shape)}")
    rows, cols = x.shape
    square = block[0] == BLOCK
    src = x.detach()
    if src.stride(1) != 1 and cols > 1:
        src = src.contiguous()
    straight = turned = None
    if orientation != "columns":
        straight = _empty_blocks(rows, cols, dtype, square, x.device)
    if orientation != "rows":
        turned = _empty_blocks(cols, rows, dtype, square, x.device)
    if x.numel():
        with device_guard(x.device):
            launcher.quantize_blocks(src.data_ptr(), _FORMATS[src.dtype], rows, cols,
                                     src.stride(0), fmt, rule, int(square), int(seed) & _MASK32,
                                     int(offset) & _MASK32, *_addresses(straight),
                                     *_addresses(turned), stream_handle(x.device))
    if orientation == "both":
        return straight, turned
    return straight if turned is None else turned


def _operand(name, t):
    """(srs_blocks, tensors to keep alive) of a BlockTensor, checked."""
    data, scale = t
    if data.dtype not in _FP8:
        raise TypeError(f"{name}: block data are float8_e4m3fn or float8_e5m2, got {data.dtype}")
    if scale.dtype != torch.float8_e8m0fnu:
        raise TypeError(f"{name}: block scales are float8_e8m0fnu, got {scale.dtype}")
    if data.dim() != 2 or scale.dim() != 2:
        raise ValueError(f"{name}: data and scale must be matrices")
    if data.device != scale.device:
        raise ValueError(f"{name}: data and scale must be on the same CUDA device")
    rows, cols = data.shape
    blocks = -(-cols // BLOCK)
    high = scale.shape[0]
    if scale.shape[1] != blocks or high not in (rows, -(-rows // BLOCK)):
        raise ValueError(f"{name}: scale of shape {tuple(scale.shape)} does not fit data of shape "
                         f"{tuple(data.shape)}")
    # The products' copies need 16-byte rows; a tensor laid out otherwise is copied once.
    if data.numel() and (data.stride(1) != 1 or data.stride(0) % 16 or data.data_ptr() % 16
                         or data.stride(0) < cols):
        padded = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.uint8, device=data.device)
        padded[:, :cols].copy_(data.view(torch.uint8))
        data = padded.view(data.dtype)
    if scale.numel() and (scale.stride(1) != 1 and blocks > 1 or scale.stride(0) < blocks):
        scale = scale.view(torch.uint8).contiguous().view(scale.dtype)
    op = _native.SrsBlocks()
    op.data, op.scale = data.data_ptr(), scale.data_ptr()
    op.rows, op.pitch, op.scale_pitch = rows, data.stride(0), scale.stride(0)
    op.format, op.square = _FP8[data.dtype], int(high != rows)
    return op, (data, scale)


def matmul_blocks(a, b, *, dtype=torch.bfloat16):
    """``a @ b.T`` of two BlockTensors (a: M x K, b: N x K), summed in FP32.

    Either operand may be E4M3 or E5M2 with scales of either block form; the
    result is FP32, BF16 or FP16.  K = 0 gives zeros."""
    if dtype not in _FORMATS:
        raise TypeError(f"matmul_blocks gives FP32, BF16 or FP16, got {dtype}")
    launcher = _native.launcher()
    device = a.data.device
    launcher.check_device(device, "matmul_blocks")
    if b.data.device != device:
        raise ValueError("all tensors must be on the same CUDA device")
    if a.data.dim() == 2 and b.data.dim() == 2 and a.data.shape[1] != b.data.shape[1]:
        raise ValueError(f"rows of different lengths: {tuple(a.data.shape)} and "
                         f"{tuple(b.data.shape)}")
    with device_guard(device):
        left, keep_a = _operand("a", a)
        right, keep_b = _operand("b", b)
        out = torch.empty((left.rows, right.rows), dtype=dtype, device=device)
        if out.numel():
            launcher.matmul_blocks(left, right, a.data.shape[1], out.data_ptr(), _FORMATS[dtype],
                                   stream_handle(device))
    del keep_a, keep_b
    return out
