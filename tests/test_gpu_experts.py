"""Products of rows in groups against FP64, expert by expert, from the blocks that
``quantize_blocks`` gives for each expert alone.

Tolerance, as for ``matmul_blocks``: FP32 sums of K exact terms are within (K + 2) * 2^-23 of
sum |a||b|, and the result's own rounding adds 2^-24, 2^-8 or 2^-11 of its size (2^-25, the
half of its smallest step, for an FP16 result below its normal range)."""

import pytest
import torch

import sr_states
from sr_states import expert_linear, quantize_blocks, quantize_stack

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
FLOOR = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}


def close(got, a, b, dtype):
    """got == a @ b.T of FP64 operands, up to the tolerance above."""
    exact, sizes = a @ b.mT, a.abs() @ b.abs().mT
    error = (a.shape[-1] + 2) * 2.0**-23 * sizes
    limit = error + HALF_ULP[dtype] * (exact.abs() + error) + FLOOR[dtype]
    assert got.dtype == dtype
    wrong = (got.double() - exact).abs() > limit
    assert not wrong.any(), (wrong.sum().item(), (got.double() - exact).abs().max().item())


def values(shape, seed, device, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    return (x * torch.exp(torch.randn((*shape[:-1], 1), generator=gen))).to(device, dtype)


def ends_of(sizes, device, dtype=torch.int32):
    return torch.tensor(sizes).cumsum(0).to(device, dtype)


def spans(sizes):
    start = 0
    for e, size in enumerate(sizes):
        yield e, slice(start, start + size)
        start += size


def dequantized(x, **how):
    got = quantize_blocks(x, **how)
    return got.dequantize().double()


SIZES = [[1], [0, 1, 0], [2, 0, 5, 1], [128], [129, 0, 127], [300, 5, 0, 700],
         [0, 0, 0], [16] * 8, [33] * 5 + [0] * 40 + [1], [1000, 3, 64]]
WIDTHS = [(128, 128), (333, 77), (64, 300), (1, 5), (1024, 257)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s))[:24])
@pytest.mark.parametrize("width", WIDTHS, ids=lambda w: f"{w[0]}x{w[1]}")
@pytest.mark.parametrize("tail", [0, 3])
def test_forward_and_gradients(sizes, width, tail, cuda_device):
    k, n = width
    rows = sum(sizes) + tail
    if rows == 0:
        rows = 2
    seed = sum(sizes) + k
    dtype = (torch.bfloat16, torch.float32, torch.float16)[(len(sizes) + k) % 3]
    grad = (E4M3, E5M2)[n % 2]
    x = values((rows, k), seed, cuda_device, dtype)
    w = values((len(sizes), n, k), seed + 1, cuda_device, dtype)
    dy = values((rows, n), seed + 2, cuda_device, dtype)
    ends = ends_of(sizes, cuda_device)
    x.requires_grad_(), w.requires_grad_()
    y = expert_linear(x, w, ends, grad_dtype=grad, seed=9)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w, y = x.detach(), w.detach(), y.detach()
    assert y.shape == (rows, n) and dx.shape == x.shape and dw.shape == w.shape
    by_row = dequantized(dy, dtype=grad, rounding="stochastic", seed=9)
    for e, s in spans(sizes):
        square = {"block": (128, 128)}
        wq = dequantized(w[e], **square)
        if s.stop == s.start:
            assert not dw[e].any()
            continue
        close(y[s], dequantized(x[s]), wq, dtype)
        close(dx[s], by_row[s], wq.mT, dtype)
        columns = dequantized(dy[s], dtype=grad, rounding="stochastic", seed=9,
                              offset=s.start * n, orientation="columns")
        close(dw[e], columns, dequantized(x[s], orientation="columns"), dtype)
    for rest in (y[sum(sizes):], dx[sum(sizes):]):
        assert not rest.any() and not rest.isnan().any()
    # kept blocks give what the call's own quantisation gives
    kept = quantize_stack(w, block=(128, 128))
    assert torch.equal(expert_linear(x, kept, ends), y)
    assert torch.equal(expert_linear(x, kept, ends.long()), y)


@pytest.mark.parametrize("square", [False, True], ids=["row", "square"])
@pytest.mark.parametrize("shape", [(1, 5, 7), (3, 128, 256), (4, 130, 77), (2, 1, 300)],
                         ids=lambda s: "x".join(map(str, s)))
def test_stacks_are_quantised_matrix_by_matrix(shape, square, cuda_device):
    block = (128, 128) if square else (1, 128)
    for source in (torch.float32, torch.bfloat16):
        x = values(shape, 3, cuda_device, source)
        for rounding in ("nearest", "stochastic"):
            for orientation in ("rows", "columns", "both"):
                how = {"block": block, "rounding": rounding, "seed": 4,
                       "orientation": orientation, "dtype": E5M2 if square else E4M3}
                got = quantize_stack(x, offset=11, **how)
                pairs = got if orientation == "both" else (got,)
                for b in range(shape[0]):
                    want = quantize_blocks(x[b], offset=11 + b * shape[1] * shape[2], **how)
                    for g, v in zip(pairs, want if orientation == "both" else (want,)):
                        assert torch.equal(g.data[b].view(torch.uint8), v.data.view(torch.uint8))
                        assert torch.equal(g.scale[b].view(torch.uint8), v.scale.view(torch.uint8))
    # dequantize of a stack
    assert torch.equal(got[0].dequantize()[0], quantize_blocks(x[0], offset=11, **how)[0]
                       .dequantize())
    turned = values((shape[0], shape[2], shape[1]), 5, cuda_device).mT  # strided
    assert torch.equal(quantize_stack(turned, block=block).data.view(torch.uint8),
                       quantize_stack(turned.contiguous(), block=block).data.view(torch.uint8))


def test_rows_of_other_experts_do_not_matter(cuda_device):
    """Infinities and NaN stay in their rows, and in their expert's gradient."""
    sizes, k, n = [70, 40, 90], 200, 150
    ends = ends_of(sizes, cuda_device)
    w = values((3, n, k), 1, cuda_device, torch.bfloat16).requires_grad_()
    clean = values((210, k), 2, cuda_device, torch.bfloat16)
    dy = values((210, n), 3, cuda_device, torch.bfloat16)

    def outputs(x, dy):
        x = x.clone().requires_grad_()
        y = expert_linear(x, w, ends, seed=2)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = outputs(clean, dy)
    dirty, dirty_dy = clean.clone(), dy.clone()
    dirty[75, 3], dirty[80] = float("nan"), float("inf")
    dirty[205:] = float("nan")   # rows of no expert
    dirty_dy[205:] = float("nan")
    got = outputs(dirty, dirty_dy)
    mine = [i for i in range(200) if i not in (75, 80)]
    assert torch.equal(got[0][mine], want[0][mine])
    assert got[0][75].isnan().all() and torch.equal(got[0][200:], torch.zeros_like(got[0][200:]))
    assert torch.equal(got[1], want[1])  # dx does not read x
    assert torch.equal(got[2][0], want[2][0]) and torch.equal(got[2][2], want[2][2])


def test_ends_that_make_no_sense_stay_inside(cuda_device):
    """Falling ends are read as their running maximum, ends past the rows as the rows."""
    k, n = 128, 96
    x = values((100, k), 1, cuda_device, torch.bfloat16).requires_grad_()
    w = values((4, n, k), 2, cuda_device, torch.bfloat16).requires_grad_()
    dy = values((100, n), 3, cuda_device, torch.bfloat16)
    results = []
    for ends, dtype in (([40, 40, 100, 100], torch.int32), ([40, 10, 2000, -5], torch.int32),
                        ([40, 10, 2**40, -2**40], torch.int64)):
        ends = torch.tensor(ends, dtype=dtype, device=cuda_device)
        y = expert_linear(x, w, ends, seed=2)
        results.append((y.detach(), *torch.autograd.grad(y, (x, w), dy)))
    for result in results[1:]:
        for got, want in zip(result, results[0]):
            assert torch.equal(got, want)


def test_strides_and_layouts(cuda_device):
    sizes, k, n = [5, 0, 40], 130, 70
    ends = ends_of(sizes, cuda_device)
    wide = values((45, 2 * k + 1), 1, cuda_device, torch.bfloat16)
    w = values((3, n, k), 2, cuda_device, torch.bfloat16)
    kept = quantize_stack(w, block=(128, 128))
    want = expert_linear(wide[:, 3:3 + k].contiguous(), kept, ends)
    assert torch.equal(expert_linear(wide[:, 3:3 + k], kept, ends), want)
    turned = wide[:, 3:3 + k].t().contiguous().t()
    assert torch.equal(expert_linear(turned, kept, ends), want)
    # data with rows off 16-byte boundaries, scales with a pitch of their own
    data = torch.empty((3, n, k), dtype=torch.uint8, device=cuda_device)
    data.copy_(kept.data.view(torch.uint8))
    scale = torch.zeros((3, 4, 9), dtype=torch.uint8, device=cuda_device)
    scale[:, :kept.scale.shape[1], :kept.scale.shape[2]] = kept.scale.view(torch.uint8)
    odd = sr_states.BlockTensor(data.view(E4M3),
                                scale[:, :kept.scale.shape[1], :kept.scale.shape[2]]
                                .view(torch.float8_e8m0fnu))
    assert torch.equal(expert_linear(wide[:, 3:3 + k], odd, ends), want)
    # one scale a row and 128 columns
    rows = quantize_stack(w)
    got = expert_linear(wide[:, 3:3 + k], rows, ends)
    for e, s in spans(sizes):
        if s.stop > s.start:
            close(got[s], dequantized(wide[s, 3:3 + k]), dequantized(w[e]), torch.bfloat16)


@pytest.mark.parametrize("rows,k,n", [(0, 64, 64), (5, 0, 64), (5, 64, 0)])
def test_sizes_of_zero(rows, k, n, cuda_device):
    x = torch.ones((rows, k), device=cuda_device, requires_grad=True)
    w = torch.ones((2, n, k), device=cuda_device, requires_grad=True)
    ends = ends_of([rows // 2, rows - rows // 2], cuda_device)
    y = expert_linear(x, w, ends)
    assert y.shape == (rows, n) and not y.any()
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not dx.any() and not dw.any()


def test_another_stream_and_captured(cuda_device):
    sizes = [40, 0, 25, 35]
    x = values((100, 256), 1, cuda_device, torch.bfloat16)
    w = values((4, 192, 256), 2, cuda_device, torch.bfloat16)
    kept, ends = quantize_stack(w, block=(128, 128)), ends_of(sizes, cuda_device)
    want = expert_linear(x, kept, ends)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = expert_linear(x, kept, ends)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = expert_linear(x, kept, ends)
    other = [0, 60, 0, 30]
    ends.copy_(ends_of(other, cuda_device))
    x.mul_(2.0)
    graph.replay()
    assert torch.equal(got, expert_linear(x, kept, ends))
    assert not got[90:].any()


def test_a_captured_training_step(cuda_device):
    """Forward and backward in one graph, with an eager graph of the same leaves alive."""
    sizes = [40, 0, 25]
    ends = ends_of(sizes, cuda_device)
    x = values((70, 256), 1, cuda_device, torch.bfloat16).requires_grad_()
    w = values((3, 192, 256), 2, cuda_device, torch.bfloat16).requires_grad_()
    dy = values((70, 192), 3, cuda_device, torch.bfloat16)

    def step():
        y = expert_linear(x, w, ends, seed=4)
        return (y, *torch.autograd.grad(y, (x, w), dy))

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


def test_the_layer_trains_and_serves(cuda_device):
    layer = sr_states.BlockExperts(3, 256, 128, seed=5, device=cuda_device)
    x = values((60, 256), 1, cuda_device, torch.bfloat16)
    ends = ends_of([20, 30, 10], cuda_device)
    y = layer(x, ends)
    y.backward(torch.ones_like(y))
    assert layer.weight.grad.shape == (3, 128, 256) and layer.calls == 1
    with torch.no_grad():
        assert torch.equal(expert_linear(x, layer.quantized(), ends), y)
    state = layer.state_dict()
    other = sr_states.BlockExperts(3, 256, 128, seed=6, device=cuda_device)
    other.load_state_dict(state)
    assert (other.seed, other.calls) == (5, 1) and torch.equal(other.weight, layer.weight)


def test_refusals(cuda_device):
    x = torch.ones((4, 32), device=cuda_device)
    w = torch.ones((2, 16, 32), device=cuda_device)
    ends = torch.tensor([2, 4], device=cuda_device)
    with pytest.raises(ValueError, match="does not fit"):
        expert_linear(x, w[:, :, :16], ends)
    with pytest.raises(ValueError, match="ends of shape"):
        expert_linear(x, w, ends[:1])
    with pytest.raises(TypeError, match="int32 or int64"):
        expert_linear(x, w, ends.float())
    with pytest.raises(ValueError, match="same CUDA device"):
        expert_linear(x, w, ends.cpu())
    with pytest.raises(TypeError, match="float8"):
        expert_linear(x, w, ends, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="FP32, BF16 or FP16"):
        expert_linear(x.double(), quantize_stack(w, block=(128, 128)), ends)
    with pytest.raises(ValueError, match="no backward pass"):
        expert_linear(x.requires_grad_(), quantize_stack(w, block=(128, 128)), ends)
    with pytest.raises(ValueError, match="three dimensions"):
        quantize_stack(x)
    with pytest.raises(ValueError, match="groups must be in"):
        sr_states.group_rows(ends, 1025)
    with pytest.raises(TypeError, match="int32 or int64"):
        sr_states.group_rows(ends.float(), 4)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sr_states.group_rows(ends.cpu(), 4)
