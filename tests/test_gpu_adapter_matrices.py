"""Adapters keep to their own tokens, whatever their matrices hold."""

import pytest
import torch

from sr_states import adapter_linear, group_rows, quantize_blocks

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


def values(shape, seed, device, dtype, size=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * size).to(device,
                                                                                        dtype)


def outputs(case, up, down):
    """The result and the gradients of x, down and up."""
    leaves = [t.clone().requires_grad_() for t in (case["x"], down, up)]
    y = adapter_linear(leaves[0], case["w"], leaves[1], leaves[2], case["groups"],
                       scale=case["scale"], seed=5)
    return (y.detach(), *torch.autograd.grad(y, leaves, case["dy"]))


def make(tokens, adapters, rank, k, n, dtype, device):
    """Tokens of all adapters and of none; adapter 1 has some wherever there is room."""
    index = torch.arange(tokens) * 7 % (adapters + 1) - 1
    if tokens > 1:
        index[tokens // 2] = 1
    index = index.to(device)
    w = quantize_blocks(values((n, k), 4, device, dtype, 0.1), block=(128, 128),
                        orientation="both")
    return {"x": values((tokens, k), 1, device, dtype), "w": w, "index": index,
            "down": values((adapters, rank, k), 2, device, dtype, k**-0.5),
            "up": values((adapters, n, rank), 3, device, dtype, 0.1),
            "groups": group_rows(index, adapters), "dy": values((tokens, n), 5, device, dtype),
            "scale": torch.linspace(0.5, 1.5, adapters, device=device)}


def check_apart(case, bad, at_up, at_down):
    """With `bad` in adapter 1's matrices, all of the other tokens and adapters is as it was, and
    adapter 1's tokens get it in the column of the place, and nowhere else."""
    index, (row, r, col) = case["index"], (at_up[0], at_up[1], at_down[1])
    clean = outputs(case, case["up"], case["down"])
    up, down = case["up"].clone(), case["down"].clone()
    up[1, row, r] = bad
    down[1, at_down[0], col] = bad
    own, rest = index == 1, index != 1
    for got, which in ((outputs(case, up, case["down"]), 0), (outputs(case, case["up"], down), 1)):
        for i in (0, 1):
            assert torch.equal(got[i][rest], clean[i][rest])
        for i in (2, 3):
            assert torch.equal(got[i][0], clean[i][0]) and torch.equal(got[i][2:], clean[i][2:])
        # a matrix's own column: of the result for `up`, of x's gradient for `down`
        one, place = got[which][own], (row, col)[which]
        if own.any():
            assert not one[:, place].isfinite().any()
            others = [c for c in range(one.shape[1]) if c != place]
            # one rounding to 16 bits each, of sums that may differ in their order
            a, b = one[:, others].double(), clean[which][own][:, others].double()
            step = torch.finfo(one.dtype).eps * a.abs().maximum(b.abs())
            assert ((a - b).abs() <= step + 1e-4 * b.abs().amax()).all()


@FORMATS
@pytest.mark.parametrize("rank", [8, 20, 64, 130])
@pytest.mark.parametrize("tokens", [200, 700])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_matrices_that_are_not_finite(tokens, rank, bad, dtype, cuda_device):
    case = make(tokens, 4, rank, 333, 410, dtype, cuda_device)
    for row, r, col in ((0, 0, 332), (409, rank - 1, 130)):
        check_apart(case, bad, (row, r), (r, col))


@FORMATS
@pytest.mark.parametrize("tokens", [300])
def test_all_matrices_but_one(tokens, dtype, cuda_device):
    """Every adapter but one full of NaN: its tokens and those of none see nothing of it."""
    case = make(tokens, 40, 16, 256, 300, dtype, cuda_device)
    clean = outputs(case, case["up"], case["down"])
    up, down = (torch.full_like(case[name], float("nan")) for name in ("up", "down"))
    up[1], down[1] = case["up"][1], case["down"][1]
    got = outputs(case, up, down)
    kept = (case["index"] == 1) | (case["index"] == -1)
    for i in (0, 1):
        assert torch.equal(got[i][kept], clean[i][kept])
        assert not got[i][~kept].isfinite().any()
    for i in (2, 3):
        assert torch.equal(got[i][1], clean[i][1])


@FORMATS
@pytest.mark.parametrize("rank", [8, 20, 64, 130])
@pytest.mark.parametrize("tokens", [1, 5, 30, 64])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_few_tokens_and_matrices_that_are_not_finite(tokens, rank, bad, dtype, cuda_device):
    case = make(tokens, 4, rank, 1333, 410, dtype, cuda_device)
    for row, r, col in ((0, 0, 1332), (409, rank - 1, 130)):
        check_apart(case, bad, (row, r), (r, col))


@FORMATS
@pytest.mark.parametrize("tokens", [3, 30, 64])
def test_few_tokens_and_all_matrices_but_one(tokens, dtype, cuda_device):
    test_all_matrices_but_one(tokens, dtype, cuda_device)


@FORMATS
@pytest.mark.parametrize("rank", [12, 40])
@pytest.mark.parametrize("k,n", [(130, 19001), (19001, 130)])
def test_wide_products_and_matrices_that_are_not_finite(k, n, rank, dtype, cuda_device):
    """More tiles than SMs: a CTA has all of k, and stores what it has added by itself."""
    case = make(40, 6, rank, k, n, dtype, cuda_device)
    check_apart(case, float("nan"), (n - 1, rank - 1), (rank - 1, k - 1))


@FORMATS
def test_a_chunk_apart_is_the_chunk(dtype, cuda_device):
    """An infinity that the low part multiplies by zero's neighbours alone: with tokens whose low
    part there is zero, nothing else of adapter 1's part is lost.  (Zero times it is NaN, in its
    column.)  The other columns of its tokens are the sum of both parts."""
    case = make(20, 3, 130, 256, 300, dtype, cuda_device)
    case["up"][1, 7, 100] = float("inf")
    h = case["scale"][1].double() * (case["x"].double() @ case["down"][1].double().mT)
    with torch.no_grad():
        y = adapter_linear(case["x"], case["w"], case["down"], case["up"], case["groups"],
                           scale=case["scale"]).double()
        none = adapter_linear(case["x"], case["w"], case["down"], torch.zeros_like(case["up"]), case["groups"]).double()
    own = case["index"] == 1
    part = h[own] @ case["up"][1].double().mT
    columns = [c for c in range(300) if c != 7]
    exact = (none[own] + part)[:, columns]
    limit = 2 * torch.finfo(dtype).eps * (exact.abs() + none[own][:, columns].abs()) + 1e-4
    assert ((y[own][:, columns] - exact).abs() <= limit).all()
    assert torch.equal(y[own][:, 7], torch.sign(h[own][:, 100]) * float("inf"))
