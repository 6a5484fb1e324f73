"""BlockLinear's bookkeeping without a GPU: what a forward pass quantises, with the quantiser and
the product replaced by plain forms that hold every value."""

import pytest
import torch

import sr_states
from sr_states import blocks


@pytest.fixture
def calls(monkeypatch):
    """[(orientation, seed), ...] of the quantisations."""
    made = []

    def quantize(x, *, orientation="rows", seed=0, **_):
        made.append((orientation, seed))
        turned = blocks.BlockTensor(x.detach().t().contiguous(), torch.ones(1))
        straight = blocks.BlockTensor(x.detach().clone(), torch.ones(1))
        return {"rows": straight, "columns": turned, "both": (straight, turned)}[orientation]

    def matmul(a, b, *, dtype):
        return (a.data.float() @ b.data.float().t()).to(dtype)

    monkeypatch.setattr(blocks, "quantize_blocks", quantize)
    monkeypatch.setattr(blocks, "matmul_blocks", matmul)
    return made


def layer(**options):
    torch.manual_seed(1)
    return sr_states.BlockLinear(8, 4, dtype=torch.float32, **options)


def test_only_what_the_backward_pass_needs_is_quantised(calls):
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    for need_x in (False, True):
        for need_w in (False, True):
            x.requires_grad_(need_x), w.requires_grad_(need_w)
            calls.clear()
            y = sr_states.block_linear(x, w)
            assert [c[0] for c in calls] == ["both" if need_w else "rows",
                                             "both" if need_x else "rows"]
            assert y.requires_grad == (need_x or need_w)
            if y.requires_grad:
                calls.clear()
                y.sum().backward()
                assert [c[0] for c in calls] == [{(True, True): "both", (True, False): "rows",
                                                  (False, True): "columns"}[need_x, need_w]]
            calls.clear()
            with torch.no_grad():
                y = sr_states.block_linear(x, w)
            assert [c[0] for c in calls] == ["rows", "rows"] and not y.requires_grad
    with torch.inference_mode():
        calls.clear()
        sr_states.block_linear(x, w)
        assert [c[0] for c in calls] == ["rows", "rows"]


def test_a_checkpointed_layer_turns_its_tokens_once(calls):
    from torch.utils.checkpoint import checkpoint

    x = torch.randn(3, 8, requires_grad=True)
    got = layer()
    plain = torch.autograd.grad(got(x).sum(), (x, got.weight))
    calls.clear()
    y = checkpoint(got, x, use_reentrant=True)
    assert [c[0] for c in calls] == ["rows", "rows"]
    y.sum().backward()
    assert [c[0] for c in calls][2:4] == ["both", "both"]
    assert torch.equal(x.grad, plain[0]) and torch.equal(got.weight.grad, plain[1])
