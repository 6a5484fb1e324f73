"""FP8 blocks: quantisation bit for bit against the CPU oracle, products and gradients
against FP64.

Tolerance of a product: FP32 sums of K exact terms are within (K + 2) * 2^-23 of
sum |a||b| (each addition rounds or truncates once), and the result's own rounding
adds 2^-24, 2^-8 or 2^-11 of its size."""

import numpy as np
import pytest
import torch

import oracle
from _support import FMT
from sr_states._hash import state_key, update_key

pytestmark = pytest.mark.gpu

FP8 = [torch.float8_e4m3fn, torch.float8_e5m2]
TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
RULES = ["nearest", "stochastic"]
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def values(shape, seed, device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    return (x * torch.exp(torch.randn((shape[0], 1), generator=gen))).to(device)


def plain(x, dtype, rule, square, seed, offset=0):
    """(bits, exponents) of x's blocks from FP64 and the oracle's cast; x: FP32 on the CPU."""
    rows, cols = x.shape
    size = np.abs(x.numpy().astype(np.float64))
    size = np.where(np.isfinite(size), size, 0.0)
    high = 128 if square else 1
    size = np.pad(size, ((0, -rows % high), (0, -cols % 128)))
    top = size.reshape(size.shape[0] // high, high, -1, 128).max((1, 3))
    k = np.zeros(top.shape, np.int64)
    some = top > 0
    # top = f * 2^e with 0.5 <= f < 1; the largest value is 0.875 * 2^9 or 2^16
    f, e = np.frexp(top[some])
    k[some] = np.maximum(e - (9 if dtype == FP8[0] else 16) + (f > 0.875), -127)
    spread = np.repeat(np.repeat(k, 128, 1)[:, :cols], high, 0)[:rows]
    with np.errstate(invalid="ignore"):
        y = np.ldexp(x.numpy().astype(np.float64), -spread).astype(np.float32)
    bits = oracle.cast(np.ascontiguousarray(y).reshape(-1), FMT[dtype], RULES.index(rule), seed,
                       offset)
    return bits.reshape(rows, cols), (k + 127).astype(np.uint8)


def bits_of(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def check(x, dtype, rule, square, orientation, seed=5, offset=0):
    from sr_states import quantize_blocks

    got = quantize_blocks(x, dtype=dtype, rounding=rule, seed=seed, offset=offset,
                          block=(128, 128) if square else (1, 128), orientation=orientation)
    got = got if orientation == "both" else (got,)
    kinds = {"rows": (0,), "columns": (1,), "both": (0, 1)}[orientation]
    x32 = x.float().cpu()
    for turned, t in zip(kinds, got):
        key = state_key(seed, turned)
        if turned:
            # scales of x.T; the data keep the counters of x
            _, k = plain(x32.t().contiguous(), dtype, "nearest", square, 0)
            spread = np.repeat(k.astype(np.int64) - 127, 128, 1)[:, :x.shape[0]]
            spread = (np.repeat(spread, 128, 0)[:x.shape[1]] if square else spread).T
            with np.errstate(invalid="ignore"):
                y = np.ldexp(x32.numpy().astype(np.float64), -spread).astype(np.float32)
            bits = oracle.cast(np.ascontiguousarray(y).reshape(-1), FMT[dtype], RULES.index(rule),
                               key, offset).reshape(x.shape).T
        else:
            bits, k = plain(x32, dtype, rule, square, key, offset)
        assert np.array_equal(bits_of(t.scale), k)
        assert np.array_equal(bits_of(t.data), bits)
        assert t.data.dtype == dtype and t.scale.dtype == torch.float8_e8m0fnu


SIZES = [(1, 1), (1, 127), (3, 128), (7, 129), (128, 128), (129, 256), (200, 333), (1000, 77),
         (511, 1024)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("dtype", FP8, ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("square", [False, True], ids=["row", "square"])
def test_blocks_match_the_oracle(size, dtype, rule, square, cuda_device):
    for source in (torch.float32, torch.bfloat16, torch.float16):
        x = values(size, sum(size)).to(source).to(cuda_device)
        check(x, dtype, rule, square, "both", offset=2**32 - 100)
    for orientation in ("rows", "columns"):
        check(x, dtype, rule, square, orientation)


@pytest.mark.parametrize("dtype", FP8, ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("square", [False, True], ids=["row", "square"])
def test_special_values(dtype, square, cuda_device):
    """Blocks of zeros, infinities, NaN, subnormals, the exact top and just above it."""
    x = values((140, 400), 3)
    x[0] = 0.0
    x[1, :128] = float("inf")
    x[2, 5], x[2, 6] = float("nan"), -float("inf")
    x[3] *= 1e-42
    x[4] = -0.0
    x[5, :128] = 0.0
    x[5, 7] = TOP[dtype]
    x[6, :128] = 0.0
    x[6, 7] = float(np.nextafter(np.float32(TOP[dtype]), np.float32(np.inf)))
    x[7] = 3.0e38
    x[8, :128] = float("nan")
    x[130:, 256:] = 0.0
    check(x.to(cuda_device), dtype, "nearest", square, "both")
    check(x.to(cuda_device), dtype, "stochastic", square, "both")


def test_strided_input_and_offsets_past_32_bits(cuda_device):
    from sr_states import quantize_blocks

    base = values((300, 700), 4, cuda_device).bfloat16()
    for view in (base[3:200, 5:300], base[::2, :256], base.t(), base.t()[1:, 7:]):
        want = quantize_blocks(view.contiguous(), orientation="both")
        got = quantize_blocks(view, orientation="both")
        for t, w in zip(got, want):
            assert np.array_equal(bits_of(t.data), bits_of(w.data))
            assert np.array_equal(bits_of(t.scale), bits_of(w.scale))
    rows = (1 << 31) // 4096 + 300
    wide = values((1, 4096), 6, cuda_device).bfloat16().expand(rows, 4096)
    t = quantize_blocks(wide)
    one = quantize_blocks(wide[:1])
    assert np.array_equal(bits_of(t.data[-1:]), bits_of(one.data))
    turned = quantize_blocks(wide, orientation="columns")
    assert np.array_equal(bits_of(turned.data[:, -1]).reshape(-1),
                          bits_of(quantize_blocks(wide[:1], orientation="columns").data).reshape(-1))


def product_case(m, n, k, da, db, sa, sb, device, seed=1):
    from sr_states import quantize_blocks

    block = {False: (1, 128), True: (128, 128)}
    a = quantize_blocks(values((m, k), seed, device), dtype=da, block=block[sa])
    b = quantize_blocks(values((n, k), seed + 1, device), dtype=db, block=block[sb])
    return a, b


def assert_product(d, a, b, dtype):
    x, y = a.dequantize().double(), b.dequantize().double()
    want, size = x @ y.t(), x.abs() @ y.abs().t()
    k = x.shape[1]
    allowed = (k + 2) * 2.0**-23 * size + HALF_ULP[dtype] * want.abs() + 1e-30
    if dtype == torch.float16:
        allowed += 2.0**-25
    assert d.dtype == dtype and d.shape == want.shape
    assert bool(((d.double() - want).abs() <= allowed).all())


PRODUCTS = [(1, 1, 1), (1, 300, 128), (3, 128, 129), (16, 1000, 512), (17, 96, 640), (64, 260, 1024),
            (100, 1, 200), (128, 128, 128), (129, 257, 513), (256, 256, 1152), (300, 1000, 64),
            (520, 777, 2049), (2048, 1536, 400)]


@pytest.mark.parametrize("size", PRODUCTS, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("pair", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_products_match_fp64(size, pair, cuda_device):
    from sr_states import matmul_blocks

    for i, dtype in enumerate((torch.bfloat16, torch.float32, torch.float16)):
        sa, sb = bool(i & 1), i == 0
        a, b = product_case(*size, FP8[pair[0]], FP8[pair[1]], sa, sb, cuda_device)
        d = matmul_blocks(a, b, dtype=dtype)
        if dtype == torch.float16:  # keep within its range
            a = a._replace(scale=(a.scale.float() * 2.0**-6).to(torch.float8_e8m0fnu))
            d = matmul_blocks(a, b, dtype=dtype)
        assert_product(d, a, b, dtype)


def test_products_of_large_tiles(cuda_device):
    from sr_states import matmul_blocks

    for m, n, k in [(4096, 4096, 1100), (3001, 5003, 640), (8192, 2048, 256)]:
        a, b = product_case(m, n, k, FP8[0], FP8[1], False, True, cuda_device)
        assert_product(matmul_blocks(a, b, dtype=torch.float32), a, b, torch.float32)
        d = matmul_blocks(a, b)
        assert torch.equal(d, matmul_blocks(a, b))


def test_scales_over_their_whole_range(cuda_device):
    """Scales of a row differ by 2^200 in a sum that FP32 still holds."""
    from sr_states import BlockTensor, matmul_blocks

    one = torch.ones(4, 512, device=cuda_device).to(FP8[0])
    exps = torch.tensor([[7, 127, 200, 100]] * 4, dtype=torch.uint8, device=cuda_device)
    back = torch.tensor([[247, 127, 54, 100]] * 4, dtype=torch.uint8, device=cuda_device)
    a = BlockTensor(one, exps.view(torch.float8_e8m0fnu))
    b = BlockTensor(one, back.view(torch.float8_e8m0fnu))
    want = 128 * (1.0 + 1.0 + 1.0 + 2.0**-54)
    d = matmul_blocks(a, b, dtype=torch.float32)
    assert bool(((d.double() - want).abs() <= 514 * 2.0**-23 * want).all())


def test_operand_layouts_and_empty_sizes(cuda_device):
    from sr_states import BlockTensor, matmul_blocks

    a, b = product_case(70, 90, 333, FP8[0], FP8[0], False, False, cuda_device)
    want = matmul_blocks(a, b)
    odd = BlockTensor(a.data.contiguous(), a.scale)  # row pitch 333
    assert odd.data.stride(0) == 333 and torch.equal(matmul_blocks(odd, b), want)
    shifted = torch.empty(70 * 336 + 1, dtype=torch.uint8, device=cuda_device)[1:].view(70, 336)
    shifted[:, :333] = a.data.view(torch.uint8)
    odd = BlockTensor(shifted.view(FP8[0])[:, :333], a.scale)
    assert torch.equal(matmul_blocks(odd, b), want)
    turned = BlockTensor(a.data.view(torch.uint8).t().contiguous().view(FP8[0]).t(),
                         a.scale.view(torch.uint8).t().contiguous().t().view(a.scale.dtype))
    assert torch.equal(matmul_blocks(turned, b), want)
    wide = torch.full((70, 9), 3, dtype=torch.uint8, device=cuda_device)
    wide[:, 2:5] = a.scale.view(torch.uint8)
    odd = BlockTensor(a.data, wide[:, 2:5].view(a.scale.dtype))
    assert torch.equal(matmul_blocks(odd, b), want)
    for m, n, k in [(0, 5, 128), (5, 0, 128), (5, 6, 0), (0, 0, 0)]:
        x, y = product_case(m, n, k, FP8[0], FP8[0], False, False, cuda_device)
        d = matmul_blocks(x, y)
        assert d.shape == (m, n) and not d.any()


def test_nan_reaches_its_row_and_column_alone(cuda_device):
    from sr_states import matmul_blocks, quantize_blocks

    x = values((40, 300), 1, cuda_device)
    x[7, 140] = float("nan")
    d = matmul_blocks(quantize_blocks(x), quantize_blocks(values((50, 300), 2, cuda_device)))
    assert d[7].isnan().all() and not d[:7].isnan().any() and not d[8:].isnan().any()


# ------------------------------------------------------------------ linear --


def test_linear_is_exact_on_representable_values(cuda_device):
    """Small integers are held exactly, so y, dx and dW are integer products, and the
    gradients equal the differences of the layer's own outputs."""
    from sr_states import block_linear

    gen = torch.Generator().manual_seed(1)
    integers = lambda *s: torch.randint(-4, 5, s, generator=gen).float().to(cuda_device)  # noqa
    x, w, dy = integers(2, 65, 300), integers(130, 300), integers(2, 65, 130)
    x.requires_grad_(), w.requires_grad_()
    y = block_linear(x, w, seed=3)
    y.backward(dy)
    assert torch.equal(y, x.detach() @ w.detach().t())
    assert torch.equal(x.grad, dy @ w.detach())
    assert torch.equal(w.grad, torch.einsum("btn,btk->nk", dy, x.detach()))
    with torch.no_grad():
        for grad, at in ((x.grad, x), (w.grad, w)):
            step = torch.zeros_like(at)
            step.view(-1)[torch.randint(0, at.numel(), (20,), generator=gen).to(cuda_device)] = 1.0
            args = (x + step, w) if at is x else (x, w + step)
            difference = ((block_linear(*args) - y) * dy).sum()
            assert float(difference) == float((grad * step).sum())


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("grad_dtype", FP8, ids=["e4m3", "e5m2"])
def test_linear_gradients_are_products_of_their_blocks(rule, grad_dtype, cuda_device):
    from sr_states import block_linear, quantize_blocks

    x = values((75, 260), 1, cuda_device).bfloat16().requires_grad_()
    w = values((200, 260), 2, cuda_device).bfloat16().requires_grad_()
    dy = (values((75, 200), 3, cuda_device) * 1e-6).bfloat16()
    y = block_linear(x, w, grad_dtype=grad_dtype, grad_rounding=rule, seed=77)
    y.backward(dy)
    square = (128, 128)
    assert_product(y.detach(), quantize_blocks(x), quantize_blocks(w, block=square),
                   torch.bfloat16)
    rows, columns = quantize_blocks(dy, dtype=grad_dtype, rounding=rule, seed=77,
                                    orientation="both")
    assert_product(x.grad, rows, quantize_blocks(w, block=square, orientation="columns"),
                   torch.bfloat16)
    assert_product(w.grad, columns, quantize_blocks(x, orientation="columns"), torch.bfloat16)
    # one gradient alone, and one that arrives as a broadcast
    for need in (x, w):
        alone = [t.detach().clone().requires_grad_(t is need) for t in (x, w)]
        block_linear(*alone, grad_dtype=grad_dtype, grad_rounding=rule, seed=77).backward(dy)
        got = alone[0 if need is x else 1].grad
        assert torch.equal(got, need.grad)
    spread = dy[:1].expand(75, 200)
    a, b = (torch.autograd.grad(block_linear(x, w, seed=5), (x, w), g)
            for g in (spread, spread.contiguous()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_stochastic_gradients_are_unbiased(cuda_device):
    """Mean of dW over 256 seeds against the product of the unrounded gradient: a
    rounding moves an element by less than one step, 1/8 of its size at most in
    E4M3, with standard deviation at most 1/16 of it; five sigma of the mean."""
    from sr_states import block_linear, quantize_blocks

    x = values((64, 128), 1, cuda_device).requires_grad_(False)
    w = values((32, 128), 2, cuda_device).requires_grad_()
    dy = values((64, 32), 3, cuda_device)
    total = torch.zeros(32, 128, dtype=torch.float64, device=cuda_device)
    for seed in range(256):
        (dw,) = torch.autograd.grad(block_linear(x, w, seed=seed), (w,), dy)
        total += dw.double()
    held = quantize_blocks(x, orientation="columns").dequantize().double()  # 128 x 64
    want = dy.double().t() @ held.t()
    top = dy.abs().amax(0).double()  # a block is one column of dy; its smallest step is 2^-15 of top
    step = torch.maximum(dy.abs().double() / 8, top * 2.0**-15)
    sigma = ((step / 2).square().t() @ held.t().square()).sqrt() / 16
    assert bool(((total / 256 - want).abs() <= 5 * sigma + 1e-5 * want.abs().max()).all())


def test_serving_form_and_module(cuda_device):
    from sr_states import BlockLinear, block_linear, matmul_blocks, quantize_blocks

    layer = BlockLinear(400, 260, seed=3, device=cuda_device)
    kept = layer.quantized()
    for tokens in (1, 2, 15, 16, 17, 40, 64, 65, 128, 200):
        x = values((tokens, 400), tokens, cuda_device).bfloat16()
        with torch.no_grad():
            y = block_linear(x, kept)
            assert torch.equal(layer(x), y)
        assert_product(y, quantize_blocks(x), kept, torch.bfloat16)
        assert torch.equal(y, matmul_blocks(quantize_blocks(x), kept))
    assert block_linear(x.view(2, 100, 400), kept).shape == (2, 100, 260)
    assert block_linear(x[:0], kept).shape == (0, 260)
    calls = layer.calls
    x.requires_grad_()
    dy = values((200, 260), 9, cuda_device).bfloat16()
    got = torch.autograd.grad(layer(x), (x, layer.weight), dy)
    want = torch.autograd.grad(block_linear(x, layer.weight, seed=update_key(3, calls + 1, 0)),
                               (x, layer.weight), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = x[:0].detach().requires_grad_()
    dx, dw = torch.autograd.grad(layer(empty), (empty, layer.weight), dy[:0])
    assert dx.shape == (0, 400) and not dw.any()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.no_grad():
        other = block_linear(x, kept)
    torch.cuda.current_stream().wait_stream(stream)
    with torch.no_grad():
        assert torch.equal(other, block_linear(x, kept))


@pytest.mark.parametrize("shape,outputs", [((0, 256), 128), ((2, 0, 256), 128), ((3, 0), 128),
                                           ((2, 3, 0), 64), ((2, 3, 256), 0), ((256,), 64),
                                           ((0,), 64)], ids=str)
def test_linear_of_vectors_and_sizes_of_zero(shape, outputs, cuda_device):
    from sr_states import block_linear, quantize_blocks

    # small integers: every block holds them exactly, and BF16 their sums below 256
    gen = torch.Generator().manual_seed(3)
    x = torch.randint(-1, 2, shape, generator=gen).to(cuda_device, torch.bfloat16)
    w = torch.randint(-1, 2, (outputs, shape[-1]), generator=gen).to(cuda_device, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    want = x.detach().double() @ w.detach().double().T
    y = block_linear(x, w)
    assert y.shape == want.shape and torch.equal(y.double(), want)
    kept = quantize_blocks(w.detach(), block=(128, 128))
    with torch.no_grad():
        assert torch.equal(block_linear(x, kept).double(), want)
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad.double(), torch.ones_like(want) @ w.detach().double())
    flat = x.detach().double().reshape(want.numel() // outputs if outputs else 6, shape[-1])
    assert torch.equal(w.grad.double(), torch.ones(
        (flat.shape[0], outputs), dtype=torch.float64, device=cuda_device).T @ flat)


def test_settings_of_the_gradient_are_refused_in_the_forward_pass(cuda_device):
    from sr_states import block_linear

    x = torch.ones((4, 128), device=cuda_device, requires_grad=True)
    w = torch.ones((128, 128), device=cuda_device)
    with pytest.raises(TypeError):
        block_linear(x, w, grad_dtype=torch.float16)
    with pytest.raises(ValueError):
        block_linear(x, w, grad_rounding="upward")


def test_refusals(cuda_device):
    from sr_states import BlockTensor, block_linear, matmul_blocks, quantize_blocks

    x = values((8, 128), 1, cuda_device)
    for bad, error in (({"dtype": torch.bfloat16}, TypeError), ({"block": (1, 64)}, ValueError),
                       ({"orientation": "none"}, ValueError), ({"rounding": "none"}, ValueError)):
        with pytest.raises(error):
            quantize_blocks(x, **bad)
    for t in (x.double(), x.int()):
        with pytest.raises(TypeError):
            quantize_blocks(t)
    for t in (x[0], x[None]):
        with pytest.raises(ValueError, match="matrix"):
            quantize_blocks(t)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_blocks(x.cpu())
    a = quantize_blocks(x)
    with pytest.raises(TypeError):
        matmul_blocks(a, a, dtype=torch.float64)
    with pytest.raises(ValueError, match="lengths"):
        matmul_blocks(a, quantize_blocks(x[:, :64]))
    with pytest.raises(TypeError):
        matmul_blocks(BlockTensor(x, a.scale), a)
    with pytest.raises(TypeError):
        matmul_blocks(BlockTensor(a.data, a.scale.view(torch.uint8)), a)
    with pytest.raises(ValueError, match="fit"):
        matmul_blocks(BlockTensor(a.data, a.scale[:3]), a)
    with pytest.raises(ValueError, match="device"):
        matmul_blocks(a, BlockTensor(a.data.cpu(), a.scale.cpu()))
    with pytest.raises(ValueError, match="backward"):
        block_linear(x.clone().requires_grad_(), a)
    with pytest.raises(ValueError, match="fit"):
        block_linear(x, quantize_blocks(x[:, :64]))


def test_no_wait_ran_out(cuda_device):
    from sr_states.cuda import _native

    assert _native.launcher().product_status() == 0
