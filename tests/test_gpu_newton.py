"""Newton-Schulz orthogonalisation and the Muon step against plain FP64 forms.

Tolerances.  FP16 rounds to within u = 2^-11 of a value.  A step rounds G, P and X
once each, a five-step run 15 matrices in all, and X_0 once more; for matrices
whose singular values lie within a few orders of magnitude the relative errors
(2-norms over the whole matrix) add up to at most 16 u = 0.8 %.  A result in FP16 or
BF16 adds its own rounding, 2^-11 or 2^-8.  One step with the coefficients
(1, 0, 0) rounds X_0 and the result of a product with the identity: 2 u."""

import math

import pytest
import torch

import oracle
from _support import FMT, from_bits, tbits
from sr_states._hash import state_key, update_key

pytestmark = pytest.mark.gpu

U = 2.0**-11
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: U}


def newton(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    a, b, c = coefficients
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT
            x = a * x + (b * g + c * g @ g) @ x
        else:
            g = x.mT @ x
            x = a * x + x @ (b * g + c * g @ g)
    return x


def relative(got, want):
    return float(torch.linalg.vector_norm(got.double() - want) / torch.linalg.vector_norm(want))


SIZES = [(1, 1, 1), (1, 1, 200), (2, 200, 1), (1, 7, 7), (3, 64, 64), (1, 127, 129), (2, 128, 128),
         (1, 130, 1000), (1, 1000, 130), (5, 333, 200), (1, 256, 256), (1, 257, 255),
         (1, 640, 2049), (12, 768, 768), (1, 2304, 768), (1, 1601, 4100)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", list(TYPES))
def test_orthogonalize_matches_fp64(size, kind, cuda_device):
    from sr_states import orthogonalize

    gen = torch.Generator().manual_seed(sum(size))
    x = (torch.randn(size, generator=gen) * 1e-3).to(TYPES[kind]).to(cuda_device)
    y = orthogonalize(x)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    assert relative(y, newton(x)) <= 16 * U + ROUNDING[y.dtype]


@pytest.mark.parametrize("size", SIZES + [(1, 2048, 2048), (2, 3000, 700)],
                         ids=lambda s: "x".join(map(str, s)))
def test_fp32_and_fp16_results_hold_more_digits(size, cuda_device):
    """Held as pairs of FP16 numbers, values keep 22 bits (or 2^-25 of a matrix's
    typical element) and products drop 2^-22 of their size, with FP32 sums (sqrt(K) *
    2^-24 over K terms, K up to 4100): 15 products and their amplification stay within
    2^-12; an FP16 result adds its own 2^-11 per element, 0.3 of it in the mean."""
    from sr_states import orthogonalize

    gen = torch.Generator().manual_seed(sum(size))
    x = (torch.randn(size, generator=gen) * 1e-3).to(cuda_device)
    want = newton(x)
    assert relative(orthogonalize(x), want) <= 2.0**-12
    assert relative(orthogonalize(x, dtype=torch.float16), want) <= 2.0**-12 + U


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1.0, 1e4, 1e30])
def test_scale_of_the_input_does_not_matter(scale, cuda_device):
    """Squares of 1e30 and 1e-30 leave FP32's range; the norm is summed in FP64."""
    from sr_states import orthogonalize

    x = torch.randn(2, 90, 200, generator=torch.Generator().manual_seed(1)).to(cuda_device) * scale
    y = orthogonalize(x, eps=0.0)
    assert relative(y, newton(x, eps=0.0)) <= 16 * U


def test_first_matrix_is_normalised_exactly_up_to_rounding(cuda_device):
    from sr_states import orthogonalize

    for shape in [(60, 100), (100, 60), (700, 300)]:
        x = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(cuda_device)
        y = orthogonalize(x, steps=1, coefficients=(1.0, 0.0, 0.0))
        assert relative(y, newton(x, 1, (1.0, 0.0, 0.0))) <= 2 * U


def test_known_result_of_orthogonal_and_diagonal_matrices(cuda_device):
    """X = Q / sqrt(n) for orthogonal Q: every step maps the one singular value s to
    a s + b s^3 + c s^5."""
    from sr_states import orthogonalize

    n = 200
    q, _ = torch.linalg.qr(torch.randn(n, n, generator=torch.Generator().manual_seed(3),
                                       dtype=torch.float64))
    s = 1.0 / math.sqrt(n)
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s**3 + 2.0315 * s**5
    y = orthogonalize(q.float().to(cuda_device)).cpu()
    assert relative(y, s * q) <= 16 * U


def test_strides_batches_and_streams(cuda_device):
    from sr_states import orthogonalize

    gen = torch.Generator().manual_seed(4)
    big = torch.randn(3, 70, 90, generator=gen).to(cuda_device)
    want = orthogonalize(big[:, 3:53, 5:80].contiguous())
    assert torch.equal(orthogonalize(big[:, 3:53, 5:80]), want)
    turned = big.transpose(1, 2)
    assert torch.equal(orthogonalize(turned), orthogonalize(turned.contiguous()))
    assert torch.equal(orthogonalize(big[1]), orthogonalize(big)[1])
    assert torch.equal(orthogonalize(big.view(3, 1, 70, 90)), orthogonalize(big).view(3, 1, 70, 90))
    assert torch.equal(orthogonalize(big[:1].expand(4, 70, 90))[3], orthogonalize(big)[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = orthogonalize(big)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, orthogonalize(big))
    for shape in [(0, 5, 5), (0, 5), (3, 0, 7), (2, 7, 0)]:
        assert orthogonalize(torch.empty(shape, device=cuda_device)).shape == shape


def test_zero_nan_and_infinite_matrices_stay_apart(cuda_device):
    from sr_states import orthogonalize

    x = torch.randn(5, 40, 70, generator=torch.Generator().manual_seed(5)).to(cuda_device)
    clean = orthogonalize(x)
    x[1] = 0.0
    x[2, 3, 4] = float("nan")
    x[3, 0, 0] = float("inf")
    y = orthogonalize(x)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[4], clean[4])
    assert not y[1].any() and y[2].isnan().all() and y[3].isnan().all()
    assert orthogonalize(x[1], eps=0.0).isnan().all()  # 0 / 0


def test_offsets_beyond_32_bits(cuda_device):
    """Results of the last matrices lie past element 2^31 of X and of the output."""
    from sr_states import orthogonalize

    x = torch.randn(1, 4096, 8192, generator=torch.Generator().manual_seed(6))
    x = x.to(cuda_device).bfloat16()
    y = orthogonalize(x.expand(66, 4096, 8192), steps=1)
    assert 65 * x.numel() > 2**31
    one = orthogonalize(x, steps=1)[0]
    assert torch.equal(y[0], one) and torch.equal(y[65], one)


def test_repeated_calls_give_the_same_bits(cuda_device):
    from sr_states import orthogonalize

    x = torch.randn(2, 500, 900, generator=torch.Generator().manual_seed(7)).to(cuda_device)
    assert torch.equal(orthogonalize(x), orthogonalize(x))


def test_refusals(cuda_device):
    from sr_states import orthogonalize

    x = torch.ones(4, 4, device=cuda_device)
    for bad in ({"steps": 0}, {"steps": 33}, {"steps": 2.0}, {"coefficients": (1.0, 2.0)},
                {"coefficients": (1.0, 2.0, float("nan"))}, {"eps": -1.0}):
        with pytest.raises(ValueError):
            orthogonalize(x, **bad)
    with pytest.raises(ValueError, match="matrices"):
        orthogonalize(x[0])
    for t in (x.double(), x.int()):
        with pytest.raises(TypeError):
            orthogonalize(t)
    with pytest.raises(TypeError):
        orthogonalize(x, dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        orthogonalize(x.cpu())


# -------------------------------------------------------------------- Muon --

STATES = [torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e5m2]


def _case(device, shapes, param, grad, state, seed=11):
    gen = torch.Generator().manual_seed(seed)
    make = lambda s, k, t: (torch.randn(s, generator=gen) * k).to(t).to(device)  # noqa: E731
    return ([make(s, 0.02, param) for s in shapes], [make(s, 1e-2, grad) for s in shapes],
            [make(s, 5e-2, state) for s in shapes])


def _want(p, g, u, lr, mom, wd, nesterov, factor):
    m, n = p.shape[0], p.numel() // p.shape[0]
    new = mom * u.double() + g.double()
    v = mom * new + g.double() if nesterov else new
    return (1 - lr * wd) * p.double() - lr * factor * newton(v.view(m, n)).view(p.shape), new


@pytest.mark.parametrize("state", STATES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_matches_fp64_and_stores_the_momentum_by_its_rule(state, param, nesterov,
                                                                     cuda_device):
    """The parameter's change is lr * s * O with |O| known to 16 u; a parameter in
    BF16 is rounded once (2^-8).  The momentum's bits are the CPU oracle's cast of
    u * momentum + g (two rounded FP32 operations)."""
    from sr_states.cuda import cuda_muon_step_

    shapes = [(64, 64), (130, 77), (64, 64), (33, 400), (8, 4, 3, 3)]
    ps, gs, us = _case(cuda_device, shapes, param, param, state)
    before = [(p.clone(), g.clone(), u.clone()) for p, g, u in zip(ps, gs, us)]
    seeds = [update_key(3, 1, i) for i in range(len(shapes))]
    cuda_muon_step_(ps, gs, us, lr=0.05, momentum_factor=0.9, weight_decay=0.1,
                    nesterov=nesterov, seeds=seeds)
    for i, (p, g, u) in enumerate(before):
        factor = max(1.0, p.shape[0] / (p.numel() // p.shape[0])) ** 0.5
        want, _ = _want(p, g, u, 0.05, 0.9, 0.1, nesterov, factor)
        change = want - 0.995 * p.double()
        off = torch.linalg.vector_norm(ps[i].double() - want)
        allowed = 16 * U * torch.linalg.vector_norm(change)
        allowed += (ROUNDING[param] + 2.0**-22) * torch.linalg.vector_norm(want)
        assert float(off) <= float(allowed), i
        new = (u.float() * 0.9 + g.float()).cpu()
        bits = oracle.cast(new.numpy().reshape(-1), FMT[state], oracle.STOCHASTIC,
                           state_key(seeds[i], 0), 0)
        expected = from_bits(bits, state).view(u.shape)
        assert (tbits(us[i]) == tbits(expected)).all(), i
        assert torch.equal(gs[i], g)


def test_muon_scale_rules(cuda_device):
    from sr_states.cuda import cuda_muon_step_

    for rule, factor in (("spectral", 2.0**0.5), ("rms", 0.2 * 200**0.5)):
        ps, gs, us = _case(cuda_device, [(200, 100)], torch.float32, torch.float32, torch.float32)
        want, _ = _want(ps[0].clone(), gs[0], us[0].clone(), 0.02, 0.95, 0.0, True, factor)
        change = torch.linalg.vector_norm(want - ps[0].double())
        cuda_muon_step_(ps, gs, us, lr=0.02, scale=rule, seeds=[1])
        assert float(torch.linalg.vector_norm(ps[0].double() - want)) <= float(16 * U * change) + 1e-6


def test_muon_optimizer_equals_its_functional_step(cuda_device):
    from sr_states import MuonSR, StateFormat
    from sr_states.cuda import cuda_muon_step_

    shapes = [(96, 160), (64, 64), (96, 160)]
    ps, gs, us = _case(cuda_device, shapes, torch.bfloat16, torch.bfloat16, torch.float8_e4m3fn)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    opt = MuonSR(params, lr=0.02, momentum=0.95, weight_decay=0.1, seed=9,
                 state_format=StateFormat(torch.float8_e4m3fn))
    us = [torch.zeros_like(u) for u in us]
    for step in (1, 2, 3):
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        cuda_muon_step_(ps, gs, us, lr=0.02, momentum_factor=0.95, weight_decay=0.1,
                        seeds=[update_key(9, step, i) for i in range(3)])
        for p, q, u in zip(params, ps, us):
            assert torch.equal(p, q)
            assert (tbits(opt.state[p]["momentum_buffer"]) == tbits(u)).all()


def test_muon_checkpoints_and_rounding_classes(cuda_device):
    from sr_states import MuonRN, MuonSR

    def run(opt, params, gs, steps):
        for _ in range(steps):
            for p, g in zip(params, gs):
                p.grad = g
            opt.step()

    shapes = [(50, 70), (70, 50)]
    ps, gs, _ = _case(cuda_device, shapes, torch.float32, torch.float32, torch.bfloat16)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    opt = MuonSR(params, seed=4)
    run(opt, params, gs, 2)
    resumed = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = MuonSR(resumed, seed=0)
    other.load_state_dict(opt.state_dict())
    run(opt, params, gs, 1)
    run(other, resumed, gs, 1)
    for p, q in zip(params, resumed):
        assert torch.equal(p, q)
        assert torch.equal(opt.state[p]["momentum_buffer"], other.state[q]["momentum_buffer"])
    nearest = [torch.nn.Parameter(p.clone()) for p in ps]
    opt = MuonRN(nearest, momentum=0.5)
    run(opt, nearest, gs, 1)
    assert torch.equal(opt.state[nearest[0]]["momentum_buffer"], gs[0].bfloat16())


def test_muon_unaligned_parameters_and_skipped_gradients(cuda_device):
    """Views that start off 16-byte boundaries take the element path, with the same bits."""
    from sr_states import MuonSR

    g = torch.randn(40 * 24 + 1, generator=torch.Generator().manual_seed(8)).to(cuda_device)
    flat = torch.zeros(2, 40 * 24 + 8, device=cuda_device)
    aligned, shifted = flat[0, 4:4 + 960].view(40, 24), flat[1, 1:961].view(40, 24)
    results = []
    for base in (aligned, shifted):
        p, idle = torch.nn.Parameter(base), torch.nn.Parameter(torch.ones(4, 4, device=cuda_device))
        p.grad = g[1:].view(40, 24) if base is shifted else g[1:].view(40, 24).clone()
        opt = MuonSR([p, idle])
        opt.step()
        assert not opt.state[idle] and bool((idle == 1).all())
        results.append((p.detach().clone(), opt.state[p]["momentum_buffer"].clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


def test_more_matrices_and_shapes_than_one_call_takes(cuda_device, monkeypatch):
    """70 matrices of one shape, 18 shapes, and a workspace limit that splits both: each
    matrix ends as it does alone."""
    from sr_states.cuda import cuda_muon_step_, muon

    shapes = [(24, 40)] * 70 + [(16 + i, 90 - i) for i in range(18)]
    ps, gs, us = _case(cuda_device, shapes, torch.bfloat16, torch.bfloat16, torch.float16)
    alone = [[t.clone() for t in (p, u)] for p, u in zip(ps, us)]
    for i, ((p, u), g) in enumerate(zip(alone, gs)):
        cuda_muon_step_([p], [g], [u], lr=0.02, seeds=[i])
    for limit in (2 << 30, 100_000):
        monkeypatch.setattr(muon, "_WORKSPACE_BYTES", limit)
        now = [[t.clone() for t in column] for column in (ps, us)]
        cuda_muon_step_(now[0], gs, now[1], lr=0.02, seeds=range(len(shapes)))
        for i, (p, u) in enumerate(alone):
            assert torch.equal(now[0][i], p) and torch.equal(now[1][i], u), (limit, i)


def test_muon_refusals(cuda_device):
    from sr_states import MuonSR
    from sr_states.cuda import cuda_muon_step_

    p, g, u = (torch.ones(8, 8, device=cuda_device) for _ in range(3))
    ok = {"lr": 0.1, "seeds": [0]}
    for bad in ({"lr": -1.0}, {"momentum_factor": 1.0}, {"weight_decay": -0.1}, {"scale": "none"},
                {"steps": 0}, {"seeds": [0, 1]}, {"formats": {"momentum_buffer": torch.float32}}):
        with pytest.raises((ValueError, TypeError)):
            cuda_muon_step_([p], [g], [u], **{**ok, **bad})
    with pytest.raises(ValueError, match="matrices"):
        cuda_muon_step_([p[0]], [g[0]], [u[0]], **ok)
    with pytest.raises(ValueError, match="overlap"):
        cuda_muon_step_([p], [g], [p], **ok)
    with pytest.raises(ValueError, match="overlap"):
        cuda_muon_step_([p, p], [g, g], [u, u.clone()], lr=0.1, seeds=[0, 1])
    with pytest.raises(ValueError, match="contiguous"):
        cuda_muon_step_([p.t()[:, :4]], [g[:, :4]], [u[:, :4]], **ok)
    with pytest.raises(TypeError):
        cuda_muon_step_([p.half()], [g], [u], **ok)
    with pytest.raises(ValueError, match="matrices"):
        MuonSR([torch.nn.Parameter(torch.ones(8, device=cuda_device))])
    for bad in ({"lr": -1.0}, {"momentum": 1.0}, {"scale": "none"}, {"ns_steps": 0}):
        with pytest.raises(ValueError):
            MuonSR([torch.nn.Parameter(p)], **bad)
    cuda_muon_step_([], [], [], lr=0.1, seeds=[])


def test_no_wait_ran_out(cuda_device):
    from sr_states.cuda import _native

    assert _native.launcher().product_status() == 0
