"""Newton-Schulz in the tiles of 256 x 256 that two CTAs share, against FP64: sizes that divide
nothing, wide and tall, results in BF16 and FP32, and Muon's update; mixed types of
parameters and gradients.

Tolerances.  Noise has all of its directions, and the three matrices rounded to FP16 in each
of five steps add up to 6 u = 6 * 2^-11 at most in the whole matrix's norm (15 independent
errors of u / sqrt(3) each and their passage through the later steps); BF16 adds half a unit in
the last place, 2^-9.  FP32 results: 2^-22 of the pairs, and FP32 sums of up to 4100
truncated terms in each product, 2^-11 in all."""

import pytest
import torch

from sr_states.cuda import _native
from test_gpu_newton import U, _case, _want, newton, relative

pytestmark = pytest.mark.gpu

BF16 = 2.0**-9


def tile(m, n, count=1, y_format=1):
    """Side of the tiles that a call with these matrices takes."""
    table = (_native.SrsMuonClass * 1)()
    table[0].count, table[0].m, table[0].n = count, m, n
    return _native.load_library().srs_newton_tile(table, 1, y_format)


PAIRS = [(3500, 3500), (2500, 4100), (4100, 2500), (3333, 3501)]


@pytest.mark.parametrize("size", PAIRS, ids=lambda s: "x".join(map(str, s)))
def test_sizes_of_cta_pairs(size, cuda_device):
    """Tiles of 256 x 256 that two CTAs share, ragged at every edge: BF16 and FP32 results."""
    from sr_states import orthogonalize

    assert tile(*size) == 256 and tile(*size, y_format=0) == 256
    gen = torch.Generator().manual_seed(7)
    x = (torch.randn(size, generator=gen) * 1e-3).to(cuda_device)
    want = newton(x)
    assert relative(orthogonalize(x, dtype=torch.bfloat16), want) <= 6 * U + BF16
    assert relative(orthogonalize(x), want) <= 2.0**-11
    x = x.bfloat16()
    assert relative(orthogonalize(x), newton(x)) <= 6 * U + BF16


@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16], ids=["g32", "g16"])
def test_muon_updates_of_cta_pairs(param, grad, cuda_device):
    from sr_states.cuda import cuda_muon_step_

    shapes = [(3333, 3501), (3501, 3333)]
    assert tile(*shapes[0]) == 256
    ps, gs, us = _case(cuda_device, shapes, param, grad, torch.float32)
    before = [(p.clone(), g.clone(), u.clone()) for p, g, u in zip(ps, gs, us)]
    cuda_muon_step_(ps, gs, us, lr=0.05, momentum_factor=0.9, weight_decay=0.1, seeds=[1, 2])
    for i, (p, g, u) in enumerate(before):
        factor = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        want, new = _want(p, g, u, 0.05, 0.9, 0.1, True, factor)
        change = torch.linalg.vector_norm(want - 0.995 * p.double())
        allowed = 6 * U * change + 2.0**-22 * torch.linalg.vector_norm(want)
        if param == torch.bfloat16:
            allowed += BF16 * torch.linalg.vector_norm(want)
        assert float(torch.linalg.vector_norm(ps[i].double() - want)) <= float(allowed), i
        assert relative(us[i], new) <= 2.0**-22


def test_mixed_types_of_parameters_and_gradients(cuda_device):
    from sr_states.cuda import cuda_muon_step_

    shapes = [(130, 77), (64, 200)]
    for param, grad in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        ps, gs, us = _case(cuda_device, shapes, param, grad, torch.bfloat16)
        before = [(p.clone(), g.clone(), u.clone()) for p, g, u in zip(ps, gs, us)]
        cuda_muon_step_(ps, gs, us, lr=0.05, momentum_factor=0.9, seeds=[1, 2])
        for i, (p, g, u) in enumerate(before):
            factor = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            want, _ = _want(p, g, u, 0.05, 0.9, 0.0, True, factor)
            change = torch.linalg.vector_norm(want - p.double())
            allowed = 16 * U * change + 2.0**-22 * torch.linalg.vector_norm(want)
            if param == torch.bfloat16:
                allowed += BF16 * torch.linalg.vector_norm(want)
            assert float(torch.linalg.vector_norm(ps[i].double() - want)) <= float(allowed), i


def test_fp32_sources_and_bf16_results(cuda_device):
    """The form of a call with dtype=torch.bfloat16, in tiles of both sides."""
    from sr_states import orthogonalize

    assert tile(128, 512) == 128 and tile(768, 768, 12) == 128 and tile(768, 768, 24) == 256
    for size in ((128, 512), (333, 1001), (24, 768, 768)):
        x = torch.randn(size, generator=torch.Generator().manual_seed(8)).to(cuda_device)
        for source in (torch.float32, torch.float16):
            y = orthogonalize(x.to(source), dtype=torch.bfloat16)
            assert relative(y, newton(x.to(source))) <= 6 * U + BF16, (size, source)


@pytest.mark.parametrize("size", [(3333, 3501), (3501, 3301), (4096, 4096)],
                         ids=lambda s: "x".join(map(str, s)))
def test_low_ranks_in_pairs(size, cuda_device):
    """What FP16 leaves of X is carried in this form, too: without it, rank 1 is 15 % off.  16 u
    for the roundings of any matrix; the sums' truncated terms, 200 k 2^-24 at most."""
    from sr_states import orthogonalize
    from sr_states.cuda import cuda_muon_step_

    m, n = size
    assert tile(m, n) == 256
    gen = torch.Generator().manual_seed(10)
    for rank in (1, 2, 40):
        x = (torch.randn(m, rank, generator=gen) @ torch.randn(rank, n, generator=gen))
        x = x.to(cuda_device)
        want = newton(x)
        cut = 200 * min(m, n) * 2.0**-24
        assert relative(orthogonalize(x, dtype=torch.bfloat16), want) <= 16 * U + BF16 + cut, rank
        assert relative(orthogonalize(x), want) <= 2.0**-12 + cut, rank
        p, u = torch.zeros_like(x), torch.zeros_like(x)
        cuda_muon_step_([p], [x], [u], lr=1.0, nesterov=False, seeds=[0])
        factor = max(1.0, m / n) ** 0.5
        assert relative(p, -factor * want) <= 16 * U + cut, rank
