"""A projection with low-rank adapters against FP64: result and gradients.

Tolerances.  With u = 2^-23 (an FP32 sum that truncates loses at most that of its terms' sizes
at each addition):

* the projection, as for ``matmul_blocks``: (K + 2) u sum |x||w|;
* the low part h = s A x: (K + 16) u |s| sum |A||x| (K terms, up to 8 parts of the sum, the
  scale); where a tensor core takes it as a pair of 16-bit numbers, 2^-17 |h| more in BF16 (each
  rounding is off by 2^-9 of what it rounds), and in FP16, whose pairs are scaled to the call's
  largest |h|, 2^-22 |h| + 2^-37 of that largest (2^-25 at 2^13 and above, or 2^-55 if the factor has
  reached its limit);
* B h: that error through |B|, and (2 rank + 8) u sum |B||h|;
* a gradient sum_t z h: the error of h through |z|, the pair's, and (2 n + 8) u sum |z||h| over
  n tokens; FP16 pairs are scaled to the adapter's largest, which leaves 2^-35 of it;
* the result's own rounding: half a step of its type.
"""

import pytest
import torch

from sr_states import (BlockTensor, RowGroups, adapter_linear, block_linear, group_rows,
                       quantize_blocks)

pytestmark = pytest.mark.gpu

U = 2.0**-23
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
FLOOR = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def values(shape, seed, device, dtype, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    return (x * torch.exp(0.5 * torch.randn((*shape[:-1], 1), generator=gen)) * size).to(device,
                                                                                         dtype)


def held(x, **how):
    return quantize_blocks(x, **how).dequantize().double()


def pair(h, dtype, largest):
    """What a pair of 16-bit numbers loses of h."""
    if dtype == torch.bfloat16:
        return 2.0**-17 * h.abs()
    return 2.0**-22 * h.abs() + 2.0**-35 * largest + 2.0**-55


def low_of(x, a, s, dtype):
    """(h, its error) of FP64 tokens and one adapter's FP64 matrix (rank x k)."""
    h, sizes = s * (x @ a.mT), abs(s) * (x.abs() @ a.abs().mT)
    return h, (a.shape[1] + 16) * U * sizes


def check(got, exact, error, dtype):
    limit = error + HALF_ULP[dtype] * (exact.abs() + error) + FLOOR[dtype]
    assert got.dtype == dtype and got.shape == exact.shape
    wrong = ~((got.double() - exact).abs() <= limit)
    assert not wrong.any(), (wrong.sum().item(), wrong.nonzero()[:4].tolist(),
                             (got.double() - exact).abs().max().item())


def expected(x, w, a, b, s, index, dtype):
    """(d, its error): d = x w^T + s (x a^T) b^T, x in FP8 blocks in the first part (`x` is
    (held, given)); a: (adapters, rank, k), b: (adapters, n, rank)."""
    inside, given = x
    exact = inside @ w.mT
    error = (w.shape[1] + 2) * U * (inside.abs() @ w.abs().mT)
    lows = [low_of(given[index == i], a[i], s[i], dtype)[0] for i in range(a.shape[0])]
    largest = max([h.abs().max() for h in lows if h.numel()], default=torch.zeros(()))
    for i in range(a.shape[0]):
        rows = index == i
        h, off = low_of(given[rows], a[i], s[i], dtype)
        off = off + pair(h, dtype, largest)
        exact[rows] += h @ b[i].mT
        error[rows] += off @ b[i].abs().mT + (2 * a.shape[1] + 8) * U * (h.abs() @ b[i].abs().mT)
    return exact, error + 4 * U * exact.abs()


def gradient(z, h, off, dtype):
    """(sum over tokens of h z^T, its error)."""
    top = h.abs().max() if h.numel() else torch.zeros((), device=z.device)
    off = off + pair(h, dtype, top)
    return (h.mT @ z, off.mT @ z.abs() + (2 * z.shape[0] + 8) * U * (h.abs().mT @ z.abs()))


def run_case(tokens, adapters, rank, k, n, dtype, device, index, grad=E4M3, size=1.0, scale=None):
    seed = tokens + 31 * rank + k
    x = values((tokens, k), seed, device, dtype).requires_grad_()
    down = values((adapters, rank, k), seed + 1, device, dtype, k**-0.5).requires_grad_()
    up = values((adapters, n, rank), seed + 2, device, dtype, 0.1).requires_grad_()
    w = values((n, k), seed + 3, device, dtype, 0.1)
    dy = values((tokens, n), seed + 4, device, dtype, size)
    s = torch.rand(adapters, generator=torch.Generator().manual_seed(seed)) + 0.5
    given = s.to(device) if scale is None else scale
    s = s.tolist() if scale is None else [scale] * adapters
    groups = group_rows(index, adapters)
    kept = quantize_blocks(w, block=(128, 128), orientation="both")
    y = adapter_linear(x, kept, down, up, groups, scale=given, grad_dtype=grad, seed=3)
    dx, da, db = torch.autograd.grad(y, (x, down, up), dy)
    x, down, up, y = x.detach(), down.detach(), up.detach(), y.detach()
    wq = kept[0].dequantize().double()
    x64, dy64, a64, b64 = x.double(), dy.double(), down.double(), up.double()
    check(y, *expected((held(x), x64), wq, a64, b64, s, index, dtype), dtype)
    by_row = held(dy, dtype=grad, rounding="stochastic", seed=3)
    check(dx, *expected((by_row, dy64), wq.mT, b64.mT, a64.mT, s, index, dtype), dtype)
    for i in range(adapters):
        rows = index == i
        h, off = low_of(x64[rows], a64[i], s[i], dtype)
        exact, error = gradient(dy64[rows], h, off, dtype)
        check(db[i], exact.mT, error.mT, dtype)
        g, off = low_of(dy64[rows], b64[i].mT, s[i], dtype)
        check(da[i], *gradient(x64[rows], g, off, dtype), dtype)
        if not rows.any():
            assert not da[i].any() and not db[i].any()
    # inference on the same blocks gives the same values
    with torch.no_grad():
        assert torch.equal(adapter_linear(x, kept[0], down, up, groups, scale=given), y)
    return x, w, down, up, groups, y


def indices(tokens, adapters, how, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    index = torch.randint(-1, adapters, (tokens,), generator=gen)
    if how == "runs":
        index = index.sort().values.flip(0)
    if how == "one":
        index = torch.full((tokens,), adapters - 1)
    if how == "none":
        index = torch.full((tokens,), -1)
    return index.to(device)


SIZES = [(1, 1, 16, 128, 128), (3, 2, 1, 77, 333), (64, 48, 16, 256, 300), (65, 3, 8, 64, 64),
         (200, 7, 12, 300, 129), (500, 5, 64, 128, 520), (300, 4, 33, 1000, 96),
         (700, 2, 128, 264, 136), (130, 2, 200, 130, 72), (1500, 3, 24, 72, 40),
         (40, 300, 4, 64, 48), (60, 3, 256, 128, 136), (64, 5, 128, 128, 1000), (17, 1024, 20, 96, 24)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("how", ["mixed", "runs", "one", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_result_and_gradients(size, how, dtype, cuda_device):
    tokens, adapters, rank, k, n = size
    index = indices(tokens, adapters, how, cuda_device)
    run_case(*size, dtype, cuda_device, index, grad=E5M2 if rank % 3 == 0 else E4M3,
             scale=2.0 if how == "one" else None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("tokens", [50, 300])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 300.0])
def test_small_and_large_gradients_keep_their_digits(dtype, tokens, size, cuda_device):
    run_case(tokens, 3, 16, 256, 200, dtype, cuda_device,
             indices(tokens, 3, "mixed", cuda_device), size=size)


def test_low_parts_beyond_fp16_fit(cuda_device):
    """An FP16 result that fits, by inner products that do not."""
    x = torch.full((70, 64), 256.0, device=cuda_device, dtype=torch.float16)
    w = torch.zeros((32, 64), device=cuda_device, dtype=torch.float16)
    down = torch.full((1, 8, 64), 16.0, device=cuda_device, dtype=torch.float16)
    up = torch.full((1, 32, 8), 2.0**-10, device=cuda_device, dtype=torch.float16)
    groups = group_rows(torch.zeros(70, dtype=torch.int32, device=cuda_device), 1)
    for tokens in (70, 9):
        plan = RowGroups(groups.order[:tokens], (groups.ends * 0 + tokens))
        with torch.no_grad():
            y = adapter_linear(x[:tokens], w, down, up, plan)
        assert (y == 256 * 16 * 64 * 8 * 2.0**-10).all()  # 2^18 inside, 2^11 out


def test_other_forms_of_the_weight(cuda_device):
    index = indices(90, 4, "mixed", cuda_device)
    x, w, down, up, groups, y = run_case(90, 4, 8, 128, 96, torch.bfloat16, cuda_device, index,
                                         scale=1.5)
    # the weight itself, with its own gradient
    w.requires_grad_(), x.requires_grad_()
    got = adapter_linear(x, w, down, up, groups, scale=1.5, seed=3)
    assert torch.equal(got.detach(), y)
    dy = values(y.shape, 9, cuda_device, torch.bfloat16)
    dx, dw = torch.autograd.grad(got, (x, w), dy)
    want = torch.autograd.grad(block_linear(x, w, seed=3), w, dy)[0]
    assert torch.equal(dw, want)
    kept = quantize_blocks(w.detach(), block=(128, 128), orientation="both")
    again = adapter_linear(x, kept, down, up, groups, scale=1.5, seed=3)
    assert torch.equal(torch.autograd.grad(again, x, dy)[0], dx)
    with torch.no_grad():
        assert torch.equal(adapter_linear(x, w, down, up, groups, scale=1.5), y)
    # without adapters in use: the projection
    none = group_rows(torch.full((90,), 7, device=cuda_device), 4)
    with torch.no_grad():
        assert torch.equal(adapter_linear(x, kept[0], down, up, none), block_linear(x, kept[0]))


def test_only_the_gradients_asked_for(cuda_device):
    index = indices(100, 3, "mixed", cuda_device)
    x, w, down, up, groups, y = run_case(100, 3, 8, 128, 96, torch.bfloat16, cuda_device, index,
                                         scale=1.0)
    kept = quantize_blocks(w, block=(128, 128), orientation="both")
    dy = values(y.shape, 9, cuda_device, torch.bfloat16)

    def grads(which, weight):
        leaves = [t.clone().requires_grad_(name in which)
                  for name, t in (("x", x), ("down", down), ("up", up))]
        out = adapter_linear(leaves[0], weight, leaves[1], leaves[2], groups, seed=3)
        return dict(zip(which, torch.autograd.grad(
            out, [t for t in leaves if t.requires_grad], dy)))

    want = grads(("x", "down", "up"), kept)
    for which in (("x",), ("down",), ("up",), ("down", "up")):
        got = grads(which, kept if "x" in which else kept[0])
        for name in which:
            assert torch.equal(got[name], want[name])


def test_tokens_of_other_adapters_do_not_matter(cuda_device):
    index = indices(300, 3, "mixed", cuda_device)
    w = values((96, 128), 1, cuda_device, torch.bfloat16)
    kept = quantize_blocks(w, block=(128, 128), orientation="both")
    down = values((3, 8, 128), 2, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    up = values((3, 96, 8), 3, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    clean = values((300, 128), 4, cuda_device, torch.bfloat16)
    dy = values((300, 96), 5, cuda_device, torch.bfloat16)
    groups = group_rows(index, 3)

    def outputs(x):
        y = adapter_linear(x, kept, down, up, groups, seed=2)
        return (y.detach(), *torch.autograd.grad(y, (down, up), dy))

    want, dirty = outputs(clean), clean.clone()
    bad = int((index == 1).nonzero()[0])
    dirty[bad, 3] = float("nan")
    none = int((index == -1).nonzero()[0])
    dirty[none] = float("inf")
    got = outputs(dirty)
    rest = [i for i in range(300) if i not in (bad, none)]
    assert torch.equal(got[0][rest], want[0][rest]) and got[0][bad].isnan().all()
    for i in (0, 2):
        assert torch.equal(got[1][i], want[1][i]) and torch.equal(got[2][i], want[2][i])
    assert got[1][1].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 40, 200, 700])
def test_large_low_parts_of_one_adapter_leave_the_others_alone(tokens, dtype, cuda_device):
    k, n, rank = 320, 400, 20
    x = values((tokens + 5, k), 1, cuda_device, dtype)
    down = values((2, rank, k), 2, cuda_device, dtype, k**-0.5)
    up = values((2, n, rank), 3, cuda_device, dtype, 0.1)
    w = quantize_blocks(values((n, k), 4, cuda_device, dtype, 0.1), block=(128, 128),
                        orientation="both")
    index = torch.zeros(tokens + 5, dtype=torch.int32, device=cuda_device)
    index[tokens // 2:tokens // 2 + 5] = 1
    dy = values((tokens + 5, n), 5, cuda_device, dtype)
    groups, results = group_rows(index, 2), []
    for size in (1.0, 2.0**40):
        scale = torch.tensor([0.7, size], device=cuda_device)
        a, b, v = (t.clone().requires_grad_() for t in (down, up, x))
        y = adapter_linear(v, w, a, b, groups, scale=scale)
        results.append((y.detach(), *torch.autograd.grad(y, (v, a, b), dy)))
    others = index == 0
    for one, two in zip(*results):
        rows = others if one.shape[0] == tokens + 5 else 0
        assert torch.equal(one[rows], two[rows])


@pytest.mark.parametrize("tokens", [40, 200])
def test_plans_that_make_no_sense_stay_inside(tokens, cuda_device):
    """Entries of the order outside the tokens, ends that fall or pass them: results are those of
    no sensible plan, but nothing outside is touched."""
    w = quantize_blocks(values((96, 128), 1, cuda_device, torch.bfloat16), block=(128, 128),
                        orientation="both")
    x = values((tokens, 128), 4, cuda_device, torch.bfloat16).requires_grad_()
    down = values((3, 8, 128), 2, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    up = values((3, 96, 8), 3, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    order = torch.arange(tokens, dtype=torch.int32, device=cuda_device)
    order[3], order[5] = -7, 2**31 - 1
    ends = torch.tensor([tokens // 2, 3, 10**6], dtype=torch.int32, device=cuda_device)
    y = adapter_linear(x, w, down, up, RowGroups(order, ends))
    torch.autograd.grad(y, (x, down, up), torch.ones_like(y))
    torch.cuda.synchronize()


def test_layouts(cuda_device):
    """Leading dimensions, strided tokens, matrices off 16-byte boundaries, turned views."""
    index = indices(96, 4, "mixed", cuda_device)
    x, w, down, up, groups, y = run_case(96, 4, 12, 130, 100, torch.bfloat16, cuda_device, index,
                                         scale=1.0)
    kept = quantize_blocks(w, block=(128, 128))
    with torch.no_grad():
        got = adapter_linear(x.reshape(4, 24, 130), kept, down, up, groups)
        assert got.shape == (4, 24, 100) and torch.equal(got.reshape(96, 100), y)
        wide = torch.zeros((96, 400), dtype=x.dtype, device=cuda_device)
        wide[:, 7:137] = x
        assert torch.equal(adapter_linear(wide[:, 7:137], kept, down, up, groups), y)
        wide[:, 200:330] = x
        assert torch.equal(adapter_linear(wide[:, 200:330], kept, down, up, groups), y)
        a = torch.empty((4, 12, 133), dtype=x.dtype, device=cuda_device)[..., 1:131]
        b = torch.empty((12, 4, 100), dtype=x.dtype, device=cuda_device).permute(1, 2, 0)
        a.copy_(down), b.copy_(up)
        assert torch.equal(adapter_linear(x, kept, a, b, groups), y)
        long = RowGroups(groups.order.long(), groups.ends.long())
        assert torch.equal(adapter_linear(x, kept, down, up, long), y)


@pytest.mark.parametrize("tokens,k,n", [(0, 64, 64), (5, 0, 64), (5, 64, 0)])
def test_sizes_of_zero(tokens, k, n, cuda_device):
    x = torch.ones((tokens, k), device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones((n, k), device=cuda_device, dtype=torch.bfloat16)
    down = torch.ones((2, 4, k), device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    up = torch.ones((2, n, 4), device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    groups = group_rows(torch.zeros(tokens, dtype=torch.int32, device=cuda_device), 2)
    y = adapter_linear(x, w, down, up, groups)
    assert y.shape == (tokens, n) and not y.any()
    for leaf, g in zip((x, down, up), torch.autograd.grad(y, (x, down, up), torch.ones_like(y))):
        assert g.shape == leaf.shape and not g.any()


@pytest.mark.parametrize("tokens", [20, 150])
def test_captured_on_another_stream(tokens, cuda_device):
    """A serving call and a training step replayed with another batch and plan, an eager graph
    of the same leaves alive."""
    x = values((tokens, 128), 1, cuda_device, torch.bfloat16).requires_grad_()
    down = values((3, 8, 128), 2, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    up = values((3, 96, 8), 3, cuda_device, torch.bfloat16, 0.1).requires_grad_()
    dy = values((tokens, 96), 5, cuda_device, torch.bfloat16)
    w = quantize_blocks(values((96, 128), 4, cuda_device, torch.bfloat16), block=(128, 128),
                        orientation="both")
    index = indices(tokens, 3, "mixed", cuda_device)
    plan = group_rows(index, 3)

    def step():
        y = adapter_linear(x, w, down, up, plan, seed=4)
        with torch.no_grad():
            served = adapter_linear(x, w[0], down, up, plan)
        return (y, served, *torch.autograd.grad(y, (x, down, up), dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager = step()
        torch.cuda.current_stream().synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    graph.replay()
    torch.cuda.synchronize()
    for g, v in zip(got, eager):
        assert torch.equal(g.detach(), v.detach())
    fresh = group_rows(indices(tokens, 3, "mixed", cuda_device, seed=8), 3)
    plan.order.copy_(fresh.order), plan.ends.copy_(fresh.ends)
    with torch.no_grad():
        x.mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    for g, v in zip(got, step()):
        assert torch.equal(g.detach(), v.detach())


def test_refusals(cuda_device):
    def make(*shape, dtype=torch.bfloat16):
        return torch.ones(shape, device=cuda_device, dtype=dtype)

    x, w, down, up = make(6, 32), make(16, 32), make(2, 4, 32), make(2, 16, 4)
    groups = group_rows(torch.zeros(6, dtype=torch.int32, device=cuda_device), 2)
    kept = quantize_blocks(w, block=(128, 128))
    bad = [
        (TypeError, "BF16 or FP16", (x.float(), kept, down.float(), up.float(), groups), {}),
        (TypeError, "in x's dtype", (x, kept, down.half(), up, groups), {}),
        (ValueError, "do not fit a projection", (x, kept, down[:, :, :16], up, groups), {}),
        (ValueError, "do not fit a projection", (x, kept, down, up[:, :, :2], groups), {}),
        (ValueError, "does not fit a weight", (make(6, 16), kept, down, up, groups), {}),
        (ValueError, "do not fit 3 adapters", (x, kept, make(3, 4, 32), make(3, 16, 4), groups), {}),
        (ValueError, "does not fit 5 tokens", (x[:5], kept, down, up, groups), {}),
        (ValueError, r"in \[1, 256\]", (x, kept, make(2, 257, 32), make(2, 16, 257), groups), {}),
        (TypeError, "scales are FP32", (x, kept, down, up, groups), {"scale": make(2)}),
        (ValueError, "scales of shape", (x, kept, down, up, groups),
         {"scale": make(3, dtype=torch.float32)}),
        (TypeError, "pair of them", (x, (kept, 1), down, up, groups), {}),
        (ValueError, "its transpose", (x, (kept, kept), down, up, groups), {}),
        (ValueError, "same CUDA device", (x, kept, down.cpu(), up, groups), {}),
        (TypeError, "float8", (x, kept, down, up, groups), {"dtype": torch.bfloat16}),
    ]
    for error, text, args, how in bad:
        with pytest.raises(error, match=text):
            adapter_linear(*args, **how)
    with pytest.raises(ValueError, match="no backward pass"):
        adapter_linear(x.requires_grad_(), kept, down, up, groups)
    assert isinstance(kept, BlockTensor)
