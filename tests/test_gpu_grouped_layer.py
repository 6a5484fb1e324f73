"""The operators on rows in groups together, as a model uses them: tokens sent to two of four
experts each through two expert layers, beside a projection with adapters, forward and backward.

The first expert layer and the projection are checked against FP64 (tolerances as in the tests of
the operators alone); the whole against the same chain captured and replayed, and for gradients in
every leaf.  The adapters' gradients are checked against differences, too: the result is linear in
`down` and in `up`, so a difference of any size is the gradient's product with it, up to the
results' rounding, half a step of their type each."""

import pytest
import torch
import torch.nn.functional as F

import sr_states
from sr_states import adapter_linear, expert_linear, group_rows, quantize_blocks

pytestmark = pytest.mark.gpu

TOKENS, WIDTH, HIDDEN, EXPERTS, TOP, ADAPTERS, RANK = 150, 256, 320, 4, 2, 3, 8


def parts(device):
    torch.manual_seed(3)
    make = lambda *s: (torch.randn(s, device=device) * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
    leaves = {
        "x": make(TOKENS, WIDTH) * WIDTH ** 0.5,
        "router": make(EXPERTS, WIDTH),
        "first": make(EXPERTS, HIDDEN, WIDTH),
        "second": make(EXPERTS, WIDTH, HIDDEN),
        "down": make(ADAPTERS, RANK, WIDTH),
        "up": make(ADAPTERS, WIDTH, RANK),
    }
    for leaf in leaves.values():
        leaf.requires_grad_()
    base = quantize_blocks(make(WIDTH, WIDTH), block=(128, 128), orientation="both")
    index = torch.arange(TOKENS, device=device) // 40 - 1  # runs; the first tokens have none
    return leaves, base, index


def layer(leaves, base, plan, seed=1):
    """Projection with adapters, then the experts' mixture around it."""
    x = adapter_linear(leaves["x"], base, leaves["down"], leaves["up"], plan, scale=0.5, seed=seed)
    weights, chosen = (x @ leaves["router"].t()).float().softmax(-1).topk(TOP)
    rows = group_rows(chosen, EXPERTS)
    token = (rows.order // TOP).long()
    sent = x[token]
    hidden = F.silu(expert_linear(sent, leaves["first"], rows.ends, seed=seed + 1))
    back = expert_linear(hidden, leaves["second"], rows.ends, seed=seed + 2)
    share = weights.reshape(-1)[rows.order.long()].to(back.dtype)
    return x + torch.zeros_like(x).index_add(0, token, back * share[:, None]), (sent, rows)


def test_the_chain_runs_forward_and_backward(cuda_device):
    leaves, base, index = parts(cuda_device)
    plan = group_rows(index, ADAPTERS)
    y, (sent, rows) = layer(leaves, base, plan)
    grads = torch.autograd.grad(y, list(leaves.values()), torch.randn_like(y))
    for leaf, grad in zip(leaves.values(), grads):
        assert grad.shape == leaf.shape and grad.isfinite().all() and grad.any()
    ends = rows.ends.tolist()
    assert ends[-1] == TOKENS * TOP and sorted(rows.order.tolist()) == list(range(TOKENS * TOP))
    # the first expert layer against FP64
    got, start = expert_linear(sent.detach(), leaves["first"].detach(), rows.ends), 0
    for e, end in enumerate(ends):
        if end > start:
            a = quantize_blocks(sent[start:end].detach()).dequantize().double()
            b = quantize_blocks(leaves["first"][e].detach(), block=(128, 128)).dequantize().double()
            exact, sizes = a @ b.t(), a.abs() @ b.abs().t()
            limit = (WIDTH + 2) * 2.0**-23 * sizes + 2.0**-8 * (exact.abs() + 2.0**-12 * sizes)
            assert ((got[start:end].double() - exact).abs() <= limit).all()
        start = end


def test_the_chain_captured_is_the_chain(cuda_device):
    """Everything but the indices' use is replayed as it ran; with other tokens it follows them."""
    leaves, base, index = parts(cuda_device)
    plan = group_rows(index, ADAPTERS)
    dy = torch.randn((TOKENS, WIDTH), device=cuda_device).to(torch.bfloat16)

    def step():
        x = adapter_linear(leaves["x"], base, leaves["down"], leaves["up"], plan, seed=1)
        rows = group_rows(index.clamp(min=0), EXPERTS)
        y = expert_linear(x, leaves["first"], rows.ends, seed=2)
        out = expert_linear(F.silu(y), leaves["second"], rows.ends, seed=3)
        used = [leaves[k] for k in ("x", "first", "second", "down", "up")]
        return (out, *torch.autograd.grad(out, used, dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        torch.cuda.current_stream().synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    with torch.no_grad():
        leaves["x"].mul_(0.7)
    graph.replay()
    torch.cuda.synchronize()
    for g, v in zip(got, step()):
        assert torch.equal(g.detach(), v.detach())


@pytest.mark.parametrize("tokens", [40, TOKENS])
def test_adapters_gradients_against_differences(tokens, cuda_device):
    leaves, base, index = parts(cuda_device)
    x, index = leaves["x"].detach()[:tokens], index[:tokens] % ADAPTERS
    plan = group_rows(index, ADAPTERS)
    c = torch.randn((tokens, WIDTH), device=cuda_device).to(torch.bfloat16)
    down, up = leaves["down"], leaves["up"]

    def result(down, up):
        return adapter_linear(x, base[0], down, up, plan)

    y = result(down, up)
    grads = torch.autograd.grad(y, (down, up), c)
    for i, leaf in enumerate((down, up)):
        # along the gradient, where the result changes most
        step = grads[i] / grads[i].float().std() * leaf.detach().float().std()
        moved = [(leaf.detach() + sign * step).to(leaf.dtype) for sign in (1, -1)]
        real = moved[0].double() - moved[1].double()  # what rounding the moved leaf left of 2 step
        with torch.no_grad():
            ends = [(result(m, up) if i == 0 else result(down, m)).double() for m in moved]
        difference = ((ends[0] - ends[1]) * c.double()).sum()
        product = (grads[i].double() * real).sum()
        limit = (2.0**-8 * (ends[0].abs() + ends[1].abs()) * c.double().abs()).sum()
        limit = limit + 2.0**-8 * (grads[i].double().abs() * real.abs()).sum()
        limit = 1.01 * limit  # the sums' own errors are some hundred times smaller than halves
        assert (difference - product).abs() <= limit
        assert product > limit  # (a factor of two would be seen)


def test_gradients_have_one_derivative(cuda_device):
    leaves, base, index = parts(cuda_device)
    plan = group_rows(index, ADAPTERS)
    ends = torch.tensor([50, 60, 60, TOKENS], device=cuda_device)
    for y in (adapter_linear(leaves["x"], base, leaves["down"], leaves["up"], plan),
              expert_linear(leaves["x"], leaves["first"], ends)):
        with pytest.raises(RuntimeError, match="first derivative only"):
            torch.autograd.grad(y.float().sum(), leaves["x"], create_graph=True)


def test_leaves_changed_in_place_are_noticed(cuda_device):
    leaves, base, index = parts(cuda_device)
    ends = torch.tensor([50, 60, 60, TOKENS], dtype=torch.int32, device=cuda_device)
    y = expert_linear(leaves["x"], leaves["first"], ends)
    ends.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


def test_checkpointed_layers(cuda_device):
    from torch.utils.checkpoint import checkpoint

    leaves, base, index = parts(cuda_device)
    plan = group_rows(index, ADAPTERS)
    used = [leaves["x"], leaves["down"], leaves["up"]]

    def run(x, down, up):
        return adapter_linear(x, base, down, up, plan, seed=4)

    c = torch.randn((TOKENS, WIDTH), device=cuda_device).to(torch.bfloat16)
    want = torch.autograd.grad(run(*used), used, c)
    got = torch.autograd.grad(checkpoint(run, *used, use_reentrant=False), used, c)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_many_small_experts(cuda_device):
    """More experts with rows than SMs, weights of a few rows."""
    torch.manual_seed(1)
    x = torch.randn((300, 130), device=cuda_device).to(torch.bfloat16)
    for experts, n in ((200, 5), (300, 77), (1000, 24)):
        w = torch.randn((experts, n, 130), device=cuda_device).to(torch.bfloat16)
        index = torch.randint(0, experts, (300,), device=cuda_device)
        rows = group_rows(index, experts)
        sent = x[rows.order.long()]
        got = expert_linear(sent, sr_states.quantize_stack(w, block=(128, 128)), rows.ends).double()
        a = quantize_blocks(sent).dequantize().double()
        b = sr_states.quantize_stack(w, block=(128, 128)).dequantize().double()
        mine = b[index[rows.order.long()]]  # (rows, n, k)
        exact = torch.einsum("rk,rnk->rn", a, mine)
        sizes = torch.einsum("rk,rnk->rn", a.abs(), mine.abs())
        limit = 132 * 2.0**-23 * sizes + 2.0**-8 * (exact.abs() + 2.0**-12 * sizes)
        assert ((got - exact).abs() <= limit).all()
