"""A captured Muon step replays its kernels with the settings of the capture."""

import pytest
import torch

from _support import tbits

pytestmark = pytest.mark.gpu


def test_a_captured_step_repeats_with_new_gradients(cuda_device):
    from sr_states.cuda import cuda_muon_step_

    gen = torch.Generator().manual_seed(1)
    shapes = [(64, 200), (130, 77)]
    make = lambda s, t: torch.randn(s, generator=gen).to(t).to(cuda_device)  # noqa: E731
    ps = [make(s, torch.bfloat16) for s in shapes]
    us = [make(s, torch.bfloat16) for s in shapes]
    gs = [make(s, torch.float32) for s in shapes]
    new = [[make(s, torch.float32) for s in shapes] for _ in range(3)]
    step = lambda p, g, u: cuda_muon_step_(p, g, u, lr=0.02, weight_decay=0.1,  # noqa: E731
                                           seeds=[5, 6])
    eager = [[t.clone() for t in column] for column in (ps, us)]
    held = [[t.clone() for t in column] for column in (ps, us)]
    step(ps, gs, us)  # first calls set kernel attributes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ps, gs, us)
    for column, start in zip((ps, us), held):
        for t, s in zip(column, start):
            t.copy_(s)
    for gradients in new:
        for g, n in zip(gs, gradients):
            g.copy_(n)
        graph.replay()
        step(eager[0], gradients, eager[1])
        for a, b in zip(ps + us, eager[0] + eager[1]):
            assert (tbits(a) == tbits(b)).all()
