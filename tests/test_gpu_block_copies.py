"""Block copies that are columns of wider buffers: what lies beside them stays as it was."""

import ctypes

import pytest
import torch

from sr_states.cuda import _native

pytestmark = pytest.mark.gpu

FENCE = 0xA5


def fenced(rows, cols, pitch, device):
    """A buffer of bytes that ends with the last row's last column, and the copy's view."""
    before = 32
    flat = torch.full((before + (rows - 1) * pitch + cols + 64,), FENCE, dtype=torch.uint8,
                      device=device)
    return flat, flat[before:].as_strided((rows, cols), (pitch, 1))


@pytest.mark.parametrize("size", [(1, 1), (3, 5), (130, 100), (64, 128), (129, 257), (200, 7),
                                  (1, 130), (255, 383)], ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("square", [False, True], ids=["row", "square"])
@pytest.mark.parametrize("orientation", ["rows", "columns", "both"])
def test_nothing_outside_the_copies_is_written(size, square, orientation, cuda_device):
    from sr_states import quantize_blocks

    rows, cols = size
    lib = _native.load_library()
    for source, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        gen = torch.Generator().manual_seed(rows + cols)
        x = torch.randn(rows, cols, generator=gen).to(source).to(cuda_device)
        want = quantize_blocks(x, block=(128, 128) if square else (1, 128),
                               orientation=orientation)
        want = want if orientation == "both" else (want,)
        address = [None, 0, None, 0] * 2
        copies = []
        turns = {"rows": (0,), "columns": (1,), "both": (0, 1)}[orientation]
        for turn, blocks in zip(turns, want):
            r, c = blocks.data.shape
            sr, sc = blocks.scale.shape
            data = fenced(r, c, 512, cuda_device)
            scale = fenced(sr, sc, sc + 3, cuda_device)
            address[4 * turn:4 * turn + 4] = [data[1].data_ptr(), 512, scale[1].data_ptr(), sc + 3]
            copies += [(data, blocks.data), (scale, blocks.scale)]
        rc = lib.srs_quantize_blocks(
            x.data_ptr(), code, rows, cols, cols, 3, 0, int(square), 0, 0, *address,
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == _native.SRS_OK, lib.srs_last_error()
        for (flat, view), expected in copies:
            assert torch.equal(view, expected.view(torch.uint8))
            view.fill_(FENCE)
            assert bool((flat == FENCE).all())
