"""Rows in groups on the sm_100a kernels: their order, and FP8 block products with one
weight a group."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .blocks import _FORMATS, _FP8, _MASK32, BlockTensor, check_blocks

MAX_GROUPS = 1024


class RowGroups(NamedTuple):
    """Rows sorted by group.

    ``order``: int32, the rows of group 0 in their order, then those of group 1, and so on, at
    last the rows of no group; ``ends``: int32, one a group: group g has
    ``order[ends[g - 1]:ends[g]]`` (from 0 for the first)."""

    order: torch.Tensor
    ends: torch.Tensor


def group_rows(index, groups) -> RowGroups:
    """Sort rows by their group, rows of one group in their order.

    ``index``: int32 or int64 on an sm_100a GPU, any shape (taken flat), at most 2^30 rows;
    values outside ``0 .. groups - 1`` (-1, say) mean no group.  ``groups``: at most 1024.
    One kernel; the host waits for nothing."""
    launcher = _native.launcher()
    launcher.check_device(index.device, "group_rows")
    return RowGroups(*launcher.group_rows(index, int(groups)))


def quantize_groups(x, ends, *, dtype, rounding="nearest", seed=0, rows=False):
    """The transposed copy of ``x`` for ``expert_gradient``; with ``rows`` (copy by rows,
    transposed copy)."""
    fmt, rule = check_blocks(dtype, rounding)
    launcher = _native.launcher()
    launcher.check_device(x.device, "expert_linear")
    got = launcher.quantize_groups(x, ends, fmt, rule, int(seed) & _MASK32, int(rows))
    return (BlockTensor(*got[:2]), BlockTensor(*got[2:])) if rows else BlockTensor(*got)


def expert_matmul(a, weight, ends, *, dtype):
    """``a[i] @ weight[e].T`` for the rows i of group e; zeros in rows of none."""
    launcher = _native.launcher()
    launcher.check_device(a.data.device, "expert_linear")
    return launcher.expert_matmul(*a, *weight, ends, _FORMATS[dtype])


def expert_blocks(x, weight, ends, dtype):
    """The same of a tensor quantised to nearest in rows and weights kept by the caller, in one
    call; the result has x's dtype."""
    launcher = _native.launcher()
    launcher.check_device(x.device, "expert_linear")
    if dtype not in _FP8:
        raise TypeError(f"blocks are held in float8_e4m3fn or float8_e5m2, got {dtype}")
    return launcher.expert_linear(x, *weight, ends, _FP8[dtype])


def expert_gradient(a_t, b_t, rows, ends, *, dtype):
    """``a_e.T @ b_e`` for every group e from the transposed copies of ``quantize_groups``."""
    launcher = _native.launcher()
    launcher.check_device(a_t.data.device, "expert_linear")
    return launcher.expert_gradient(*a_t, *b_t, rows, ends, _FORMATS[dtype])


class Low(NamedTuple):
    """The low part of an ``adapter_product`` (FP32, tokens in their groups' order), and what the
    sums over it need."""

    values: torch.Tensor
    largest: torch.Tensor | None


def adapter_product(x, weight, down, up, groups, *, scale, dtype, rounding="nearest", seed=0,
                    turned=False, keep=False):
    """(``x @ weight.T`` in FP8 blocks plus the adapters' part, Low); ``turned``: x is the
    gradient of the result.  ``weight`` None: the low part alone."""
    fmt, rule = check_blocks(dtype, rounding)
    launcher = _native.launcher()
    launcher.check_device(x.device, "adapter_linear")
    scale, factor = (scale, 1.0) if isinstance(scale, torch.Tensor) else (None, float(scale))
    w, w_scale = (None, None) if weight is None else weight
    out, low, largest = launcher.adapter_linear(
        x, fmt, rule, int(seed) & _MASK32, w, w_scale, down, up, scale, factor, groups.order,
        groups.ends, int(turned), int(keep))
    return out, Low(low, largest)


def adapter_gradient(z, low, groups, *, turned=False):
    """Sums over each adapter's tokens of low by z (rank x columns), or turned."""
    launcher = _native.launcher()
    launcher.check_device(z.device, "adapter_linear")
    return launcher.adapter_gradient(z, low.values, low.largest, groups.order, groups.ends,
                                     int(turned))
