"""The operators on rows in groups as programs use them beside one another: several streams and
threads, graphs of one memory pool, saved tensors moved away, experts that hold what is not finite."""

import threading

import pytest
import torch

from sr_states import (adapter_linear, block_linear, expert_linear, group_rows, quantize_blocks,
                       quantize_stack)

pytestmark = pytest.mark.gpu


def values(shape, seed, device, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * size).to(device, torch.bfloat16)


def job(tokens, seed, device):
    """A call of each kind, forward and backward, on inputs of its own."""
    x = values((tokens, 256), seed, device).requires_grad_()
    down = values((5, 16, 256), seed + 1, device, 0.1).requires_grad_()
    up = values((5, 320, 16), seed + 2, device, 0.1).requires_grad_()
    experts = values((4, 192, 320), seed + 3, device, 0.1).requires_grad_()
    w = quantize_blocks(values((320, 256), seed + 4, device, 0.1), block=(128, 128),
                        orientation="both")
    kept = quantize_stack(experts.detach(), block=(128, 128))
    index = torch.arange(tokens, device=device) * 5 % 6 - 1
    dy = values((tokens, 192), seed + 5, device)

    def run():
        plan = group_rows(index, 5)
        y = adapter_linear(x, w, down, up, plan, seed=seed)
        sent = group_rows(index, 4)
        z = expert_linear(y[sent.order.long()], experts, sent.ends, seed=seed)
        grads = torch.autograd.grad(z, (x, down, up, experts), dy)
        with torch.no_grad():
            served = expert_linear(y[sent.order.long()], kept, sent.ends)
        return (plan.order, y.detach(), z.detach(), served, *grads)

    return run


def same(a, b):
    return all(torch.equal(u, v) for u, v in zip(a, b))


def test_streams_and_threads(cuda_device):
    jobs = [job(tokens, 10 * i, cuda_device) for i, tokens in enumerate((3, 40, 64, 200, 700))]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * len(jobs), []

    def work(i):
        try:
            stream = torch.cuda.Stream(cuda_device)
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = jobs[i]()
                    if not same(got[i], want[i]):
                        raise AssertionError(f"job {i} differs beside the others")
            stream.synchronize()
        except BaseException as error:  # noqa: BLE001 (for the main thread)
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(60)
    assert not errors, errors


def test_graphs_of_one_pool(cuda_device):
    """Two captures in one memory pool, replayed in turn: each has its own results."""
    jobs = [job(40, 1, cuda_device), job(300, 2, cuda_device)]
    want = [tuple(t.clone() for t in run()) for run in jobs]
    stream, graphs, results = torch.cuda.Stream(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for run in jobs:
            run()
        stream.synchronize()
        pool = torch.cuda.graph_pool_handle()
        for run in jobs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, pool=pool):
                results.append(run())
            graphs.append(graph)
    for which in (0, 1, 1, 0):
        graphs[which].replay()
        torch.cuda.synchronize()
        assert same(results[which], want[which])


def test_saved_tensors_moved_away_and_used_twice(cuda_device):
    x = values((90, 128), 1, cuda_device).requires_grad_()
    w = values((96, 128), 2, cuda_device).requires_grad_()
    down = values((3, 12, 128), 3, cuda_device, 0.1).requires_grad_()
    up = values((3, 96, 12), 4, cuda_device, 0.1).requires_grad_()
    experts = values((3, 64, 96), 5, cuda_device, 0.1).requires_grad_()
    plan = group_rows(torch.arange(90, device=cuda_device) // 30, 3)
    dy = values((90, 64), 6, cuda_device)
    leaves = (x, w, down, up, experts)

    def forward():
        y = adapter_linear(x, w, down, up, plan, seed=1)
        return expert_linear(y, experts, plan.ends, seed=2)

    want = torch.autograd.grad(forward(), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        z = forward()
    assert same(torch.autograd.grad(z, leaves, dy, retain_graph=True), want)
    assert same(torch.autograd.grad(z, leaves, dy), want)
    z = torch.utils.checkpoint.checkpoint(forward, use_reentrant=False)
    assert same(torch.autograd.grad(z, leaves, dy), want)


@pytest.mark.parametrize("rows", [60, 900])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_experts_and_rows_that_are_not_finite(bad, rows, cuda_device):
    """What one expert's weights or rows hold stays with them; rows of none reach nothing."""
    x, w = values((rows, 200), 1, cuda_device), values((4, 150, 200), 2, cuda_device)
    dy = values((rows, 150), 3, cuda_device)
    ends = torch.tensor([rows // 5, rows // 2, rows // 2, rows - 7], device=cuda_device)
    own = torch.zeros(rows, dtype=torch.bool, device=cuda_device)
    own[rows // 5:rows // 2] = True  # expert 1

    def run(x, w, dy):
        x, w = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = expert_linear(x, w, ends, seed=3)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    clean = run(x, w, dy)
    odd_x, odd_w, odd_dy = x.clone(), w.clone(), dy.clone()
    odd_x[rows // 5] = bad
    odd_x[rows - 3:] = bad
    odd_dy[rows // 2 - 1] = bad
    odd_dy[rows - 3:] = bad
    odd_w[1] = bad
    odd_w[2] = bad  # has no rows
    for args in ((odd_x, w, dy), (x, odd_w, dy), (x, w, odd_dy)):
        y, dx, dw = run(*args)
        assert torch.equal(y[~own], clean[0][~own]) and torch.equal(dx[~own], clean[1][~own])
        for e in (0, 2, 3):
            assert torch.equal(dw[e], clean[2][e])
    # a row's own: NaN is kept, an infinity saturates as in one layer of the row alone
    if bad != bad:
        assert run(odd_x, w, dy)[0][rows // 5].isnan().all()
    alone = block_linear(odd_x[own], w[1])
    assert torch.equal(run(odd_x, w, dy)[0][own].isnan(), alone.isnan())
