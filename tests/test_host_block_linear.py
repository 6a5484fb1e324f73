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


def draws(calls, got, count, x):
    """Seeds of the gradient roundings of the next training calls."""
    seeds = []
    for _ in range(count):
        calls.clear()
        got(x).sum().backward()
        seeds.append(calls[2][1])
    return seeds


def test_a_checkpoint_carries_the_draws(calls, tmp_path):
    x = torch.randn(3, 8)
    one, two = layer(seed=7), layer(seed=7)
    want = draws(calls, one, 5, x)
    assert len(set(want)) == 5
    assert draws(calls, two, 2, x) == want[:2]
    with torch.no_grad():
        two(x)  # evaluation draws nothing
    path = tmp_path / "layer.pt"
    torch.save(torch.nn.Sequential(two).state_dict(), path)
    resumed = torch.nn.Sequential(layer(seed=99))
    resumed.load_state_dict(torch.load(path, weights_only=True))
    assert resumed[0].seed == 7 and resumed[0].calls == 2
    assert draws(calls, resumed, 3, x) == want[2:]
    assert draws(calls, two, 3, x) == want[2:]


def test_a_state_dict_of_the_weight_alone_still_loads():
    one, two = layer(seed=3), layer(seed=4)
    two.load_state_dict({"weight": one.weight.detach()})
    assert torch.equal(one.weight, two.weight) and (two.seed, two.calls) == (4, 0)
    assert not two.load_state_dict({"weight": one.weight.detach()}, strict=False).missing_keys
    with pytest.raises(RuntimeError, match="weight"):
        two.load_state_dict({})


def test_layers_and_ranks_draw_apart(calls, monkeypatch):
    x = torch.randn(3, 8)
    first = [draws(calls, layer(), 1, x)[0] for _ in range(4)]
    assert len(set(first)) == 4
    ranks = []
    monkeypatch.setattr(torch.distributed, "is_initialized", lambda: True)
    for rank in range(4):
        monkeypatch.setattr(torch.distributed, "get_rank", lambda: rank)
        ranks.append(draws(calls, layer(seed=5), 1, x)[0])
    assert len(set(ranks)) == 4
    monkeypatch.undo()


def test_the_draws_of_a_given_seed_are_those_of_the_functional_form(calls):
    from sr_states._hash import update_key

    got = layer(seed=3)
    assert draws(calls, got, 2, torch.randn(3, 8)) == [update_key(3, 1, 0), update_key(3, 2, 0)]
