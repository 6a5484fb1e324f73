"""Rows sorted by group, against a plain stable sort: whole numbers, equal throughout."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(index, groups):
    index = index.reshape(-1)
    kept = np.where((index >= 0) & (index < groups), index, groups)
    order = np.argsort(kept, kind="stable")
    return order, np.cumsum(np.bincount(kept, minlength=groups + 1))[:groups]


def check(index, groups, device):
    from sr_states import group_rows

    got = group_rows(torch.from_numpy(index).to(device), groups)
    order, ends = plain(index, groups)
    assert got.order.dtype == got.ends.dtype == torch.int32
    assert np.array_equal(got.order.cpu().numpy(), order)
    assert np.array_equal(got.ends.cpu().numpy(), ends)


# around a warp's batch, one CTA's rows (4096) and a cluster's
ROWS = [0, 1, 31, 32, 33, 1000, 4096, 4097, 10007, 65536, 300001]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("groups", [1, 2, 31, 64, 257, 1024])
def test_rows_are_sorted_stably(rows, groups, cuda_device):
    rng = np.random.default_rng(rows * 2000 + groups)
    index = rng.integers(-2, groups + 3, rows)
    check(index.astype(np.int32), groups, cuda_device)
    check(index.astype(np.int64), groups, cuda_device)


@pytest.mark.parametrize("rows", [777, 20000])
def test_uneven_groups(rows, cuda_device):
    rng = np.random.default_rng(rows)
    for index in (np.full(rows, 5), np.full(rows, -1), np.arange(rows) % 9,
                  np.arange(rows)[::-1] // 100, np.sort(rng.integers(0, 64, rows)),
                  np.minimum(rng.geometric(0.3, rows), 63), np.full(rows, 2**31 - 1)):
        check(index.astype(np.int32), 64, cuda_device)
    wide = rng.integers(0, 64, rows) + 2**32 * rng.integers(0, 2, rows)  # the high half counts
    check(wide, 64, cuda_device)


def test_shapes_and_views(cuda_device):
    index = np.random.default_rng(1).integers(0, 8, (50, 6))
    check(index, 8, cuda_device)
    from sr_states import group_rows

    t = torch.from_numpy(index).to(cuda_device)
    got, want = group_rows(t[:, 1:4], 8), plain(index[:, 1:4], 8)
    assert np.array_equal(got.order.cpu().numpy(), want[0])


def test_a_captured_sort_follows_its_input(cuda_device):
    from sr_states import group_rows

    index = torch.zeros(500, dtype=torch.int32, device=cuda_device)
    group_rows(index, 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = group_rows(index, 16)
    for seed in range(3):
        fresh = np.random.default_rng(seed).integers(-1, 16, 500).astype(np.int32)
        index.copy_(torch.from_numpy(fresh))
        graph.replay()
        order, ends = plain(fresh, 16)
        assert np.array_equal(got.order.cpu().numpy(), order)
        assert np.array_equal(got.ends.cpu().numpy(), ends)
