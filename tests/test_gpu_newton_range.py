"""Newton-Schulz over the matrices it meets in earnest: low ranks, falling spectra, norms
far below eps and large coefficients.

Tolerances.  A BF16 result (and Muon's update) comes from G, P and X held in FP16, each
rounded to within u = 2^-11 of its elements: 15 matrices in a run of five steps, 16 u
in all, whatever the singular values are: directions that the matrix does not have are
multiplied by 3.4445 a step, so X has to be carried with more digits than FP16 until the last
of them.  The result's own rounding adds half a unit in its last place, 2^-9 of an element at
most."""

import pytest
import torch

from test_gpu_newton import U, _case, _want, newton, relative

pytestmark = pytest.mark.gpu

BF16 = 2.0**-9


def spectrum(m, n, values, gen):
    """An m x n matrix with the given singular values."""
    k = len(values)
    left, _ = torch.linalg.qr(torch.randn(m, k, generator=gen, dtype=torch.float64))
    right, _ = torch.linalg.qr(torch.randn(n, k, generator=gen, dtype=torch.float64))
    return (left * values) @ right.T


def matrices(m, n, seed=1):
    """Low ranks, falling spectra, few rows, few columns and one large element."""
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    small = min(m, n)
    found = {f"rank {r}": normal(m, r) @ normal(r, n) for r in (1, 2, 8, min(64, small))}
    for p in (1.0, 2.0, 4.0):
        found[f"k^-{p:.0f}"] = spectrum(m, n, torch.arange(1, small + 1).double() ** -p, gen)
    found["eight decades"] = spectrum(m, n, torch.logspace(0, -8, small, dtype=torch.float64), gen)
    few = torch.zeros(m, n, dtype=torch.float64)
    few[: min(4, m)] = normal(min(4, m), n)
    found["four rows"] = few
    few = torch.zeros(m, n, dtype=torch.float64)
    few[:, : min(3, n)] = normal(m, min(3, n))
    found["three columns"] = few
    found["one element"] = 1e-6 * normal(m, n)
    found["one element"][m // 2, n // 3] = 1.0
    return found


SIZES = [(16, 64), (64, 512), (512, 64), (256, 1000), (768, 768), (1000, 256), (500, 2050)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("source", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_low_ranks_and_falling_spectra(size, source, cuda_device):
    from sr_states import orthogonalize

    for name, x in matrices(*size).items():
        x = x.to(source).to(cuda_device)
        off = relative(orthogonalize(x, dtype=torch.bfloat16), newton(x))
        assert off <= 16 * U + BF16, (name, off)


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_fp32_results_of_low_ranks_and_falling_spectra(size, cuda_device):
    """Pairs of FP16 numbers leave 2^-22 of an element, 2^-12 after the amplification.  The
    tensor core truncates: each of the k terms of a sum takes up to 2^-24 of it, all of one
    sign, and the steps that follow multiply what the first ones lose by 3.4445^4 + 3.4445^3
    + ... < 200."""
    from sr_states import orthogonalize

    for name, x in matrices(*size).items():
        x = x.float().to(cuda_device)
        off = relative(orthogonalize(x), newton(x))
        assert off <= 2.0**-12 + 200 * min(size) * 2.0**-24, (name, off)


@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_muon_updates_of_low_rank_gradients(param, cuda_device):
    """The first step of a run: no momentum, gradients of few tokens."""
    from sr_states.cuda import cuda_muon_step_

    for shape in ((256, 700), (700, 256)):
        for name, g in matrices(*shape).items():
            g = g.float().to(cuda_device)
            p, u = torch.zeros(shape, dtype=param, device=cuda_device), torch.zeros_like(g)
            cuda_muon_step_([p], [g], [u], lr=1.0, seeds=[0])
            want, _ = _want(torch.zeros_like(g), g, torch.zeros_like(g), 1.0, 0.95, 0.0, True,
                            max(1.0, shape[0] / shape[1]) ** 0.5)
            off = relative(p, want)
            assert off <= 16 * U + (BF16 if param == torch.bfloat16 else 0.0), (shape, name, off)


@pytest.mark.parametrize("ratio", [1e-1, 1e-3, 1e-6, 1e-12, 1e-25])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_norms_below_eps(ratio, dtype, cuda_device):
    """X_0 = x / (|x| + eps) is then small, and keeps its digits."""
    from sr_states import orthogonalize

    gen = torch.Generator().manual_seed(5)
    for shape in ((60, 100), (300, 40)):
        x = torch.randn(shape, generator=gen).to(cuda_device)
        x *= ratio / torch.linalg.matrix_norm(x)
        off = relative(orthogonalize(x, eps=1.0, dtype=dtype), newton(x, eps=1.0))
        assert off <= 16 * U + (BF16 if dtype == torch.bfloat16 else 0.0), (shape, off)


def test_muon_steps_of_vanishing_gradients(cuda_device):
    """Gradients far below eps move a parameter by 485 times their share of it."""
    from sr_states.cuda import cuda_muon_step_

    gen = torch.Generator().manual_seed(9)
    for ratio in (1e-4, 1e-9):
        g = torch.randn(80, 130, generator=gen).to(cuda_device)
        g *= ratio * 1e-7 / torch.linalg.matrix_norm(g)
        p, u = torch.zeros_like(g), torch.zeros_like(g)
        cuda_muon_step_([p], [g], [u], lr=1.0, seeds=[0])
        want, _ = _want(torch.zeros_like(g), g, torch.zeros_like(g), 1.0, 0.95, 0.0, True, 1.0)
        assert relative(p, want) <= 16 * U


@pytest.mark.parametrize("a", [100.0, 300.0, 1e5])
def test_large_coefficients(a, cuda_device):
    """One step with G's part zero: P = a I, beyond FP16's range in part."""
    from sr_states import orthogonalize

    x = torch.randn(50, 90, generator=torch.Generator().manual_seed(6)).to(cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        y = orthogonalize(x, steps=1, coefficients=(a, 0.0, 0.0), dtype=dtype)
        assert relative(y, newton(x, 1, (a, 0.0, 0.0))) <= 3 * U + (
            BF16 if dtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("coefficients", [(400.0, -500.0, 150.0), (-300.0, 900.0, -300.0),
                                          (3.0, 2000.0, 0.0), (2.0, 0.0, 1e4)], ids=str)
def test_steps_of_large_coefficients(coefficients, cuda_device):
    """One step whose P has eigenvalues beyond 255 in places."""
    from sr_states import orthogonalize

    for name, x in matrices(60, 130).items():
        x = x.float().to(cuda_device)
        want = newton(x, 1, coefficients)
        assert relative(orthogonalize(x, steps=1, coefficients=coefficients,
                                      dtype=torch.bfloat16), want) <= 16 * U + BF16, name
