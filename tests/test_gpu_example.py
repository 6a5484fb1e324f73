"""The low-precision training example learns, repeats itself and serves what it learned."""

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLES = Path(__file__).resolve().parents[1] / "examples"


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(EXAMPLES))
    import train_low_precision

    return train_low_precision


def test_training_learns_repeats_and_serves(example, cuda_device):
    model, losses = example.train(60, cuda_device)
    # From ln(512) = 6.24 for a uniform guess; 5 % of the steps jump anywhere.
    assert losses[0] > 5.5 and losses[-1] < 3.0
    _, again = example.train(3, cuda_device)
    assert again == losses[:3]
    walk = torch.randperm(example.VOCAB, generator=torch.Generator().manual_seed(12345))
    start = torch.arange(0, 400, 25, device=cuda_device)[:, None].expand(-1, 3).contiguous()
    start[:, 1] = walk[start[:, 0].cpu()].to(cuda_device)
    start[:, 2] = walk[start[:, 1].cpu()].to(cuda_device)
    got = example.serve(model, start, 1)[:, 3].cpu()
    assert (got == walk[start[:, 2].cpu()]).float().mean() > 0.5


def test_two_streams_at_once(cuda_device):
    """Orthogonalisations on two streams (cooperative grids) give the single-stream bits."""
    from sr_states import orthogonalize

    x = [torch.randn(2, 300, 700, generator=torch.Generator().manual_seed(i)).to(cuda_device)
         for i in range(2)]
    want = [orthogonalize(t) for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(orthogonalize(x[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_calls_replay_in_a_cuda_graph(cuda_device):
    from sr_states import block_linear, orthogonalize, quantize_blocks

    x = torch.randn(100, 260, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    w = quantize_blocks(torch.randn(384, 260, generator=torch.Generator().manual_seed(2))
                        .to(cuda_device), block=(128, 128))
    call = lambda: (orthogonalize(x), block_linear(x, w), block_linear(x[:1], w))  # noqa: E731
    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        x.copy_(torch.randn(100, 260, generator=torch.Generator().manual_seed(3)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))
