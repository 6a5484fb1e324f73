"""Rows in groups on the sm_100a kernels: their order."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native


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
