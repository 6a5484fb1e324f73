"""Matrices too large for the kernels are refused before any of a step's calls is made."""

import pytest
import torch

from sr_states.cuda import _native, muon
from sr_states.cuda._tables import Update


class Shape:
    """What the planning of a step reads of a matrix."""

    def __init__(self, *shape):
        self.tensors = (self,)
        self.shape, self.numel = shape, shape[0] * shape[1]


@pytest.mark.parametrize("shape", [(1 << 25, 2), (2, 1 << 25), (1 << 17, 1 << 16)])
def test_oversized_matrices_are_refused_while_the_step_is_planned(shape):
    launcher = _native.launcher()
    updates = [Shape(64, 64), Shape(*shape), Shape(64, 96)]
    with pytest.raises(ValueError, match="too large"):
        for call in muon._calls(muon._shape_classes(updates), launcher):
            table = (_native.SrsMuonClass * len(call))()
            for entry, (m, n, chosen) in zip(table, call):
                entry.count, entry.m, entry.n = len(chosen), m, n
            launcher.muon_workspace(table)


def test_workspaces_of_sizes_that_fit():
    launcher = _native.launcher()
    table = (_native.SrsMuonClass * 1)()
    table[0].count, table[0].m, table[0].n = 3, 100, 200
    assert launcher.muon_workspace(table) > 0
    table[0].count = 65
    with pytest.raises(ValueError, match="at most 64"):
        launcher.muon_workspace(table)


def test_a_whole_step_is_refused_before_its_first_launch(monkeypatch):
    launched = []
    monkeypatch.setattr(muon, "_WORKSPACE_BYTES", 1)  # a call for each matrix

    class Launcher(_native.NativeLauncher):
        def muon_multi(self, *args):
            launched.append(args)

    def matrix(*shape):
        x = torch.empty(shape, device="meta")
        return Update((x, x, x), 0, x.numel(), 0, None)

    previous = _native.set_launcher(Launcher())
    try:
        with pytest.raises(ValueError, match="too large"):
            muon.muon_launch([matrix(64, 64), matrix(1 << 25, 2)], (0, 0), lr=0.1, momentum=0.9,
                             weight_decay=0.0, nesterov=True, scale="spectral", newton=None,
                             rng=None)
    finally:
        _native.set_launcher(previous)
    assert not launched
