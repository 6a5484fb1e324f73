"""A wait that ran out inside a product kernel reaches the caller as an error, once.

No kernel is made to wait: the word that they would write is set from the host."""

import pytest
import torch

from sr_states.cuda import _native, check_products

pytestmark = pytest.mark.gpu


@pytest.fixture
def word(cuda_device):
    found = _native.launcher().product_status_word()
    assert found.contents.value == 0
    yield found
    found.contents.value = 0


def calls(device):
    from sr_states import MuonSR, block_linear, matmul_blocks, orthogonalize, quantize_blocks

    x = torch.randn(100, 260, generator=torch.Generator().manual_seed(1)).to(device)
    w = quantize_blocks(torch.randn(384, 260, generator=torch.Generator().manual_seed(2))
                        .to(device), block=(128, 128))
    p = torch.nn.Parameter(torch.zeros(40, 60, device=device))
    p.grad = torch.randn(40, 60, generator=torch.Generator().manual_seed(3)).to(device)
    opt = MuonSR([p])
    opt.step()
    with torch.no_grad():
        block_linear(x, w)
    return p, opt, {
        "orthogonalize": lambda: orthogonalize(x),
        "matmul": lambda: matmul_blocks(quantize_blocks(x), w),
        "linear": lambda: block_linear(x, w),
        "one token": lambda: block_linear(x[:1], w),
        "muon": opt.step,
    }


def test_the_next_call_raises_and_enqueues_nothing(word, cuda_device):
    p, opt, todo = calls(cuda_device)
    for name, call in todo.items():
        torch.cuda.synchronize()
        before = p.detach().clone(), opt.state[p]["momentum_buffer"].clone()
        word.contents.value = 0x80
        with pytest.raises(RuntimeError, match="0x80"):
            call()
        assert word.contents.value == 0, name
        assert torch.equal(p, before[0]), name
        assert torch.equal(opt.state[p]["momentum_buffer"], before[1]), name
        call()


def test_checks_that_wait(word, cuda_device):
    _, opt, todo = calls(cuda_device)
    check_products(cuda_device)
    word.contents.value = 0x10000
    with pytest.raises(RuntimeError, match="0x10000"):
        check_products(cuda_device)
    check_products(cuda_device)
    word.contents.value = 0x20000
    with pytest.raises(RuntimeError, match="0x20000"):
        opt.state_dict()
    assert opt.state_dict()["state"]
    word.contents.value = 5
    assert _native.launcher().product_status() == 5
    assert _native.launcher().product_status() == 0
    for call in todo.values():
        call()
    check_products(cuda_device)
