"""Operators on rows in groups without a GPU: refusals of the C entry points before any CUDA call,
refusals of the Python calls, sizes, and the layers' bookkeeping."""

import ctypes

import pytest
import torch

import sr_states
from sr_states.cuda import _native

BAD = _native.SRS_ERR_INVALID_ARGUMENT


class Blocks(ctypes.Structure):
    _fields_ = [("data", ctypes.c_uint64), ("scale", ctypes.c_uint64), ("rows", ctypes.c_int64),
                ("pitch", ctypes.c_int64), ("scale_pitch", ctypes.c_int64),
                ("format", ctypes.c_int32), ("square", ctypes.c_int32)]


class Copy(ctypes.Structure):
    _fields_ = [("data", ctypes.c_uint64), ("scale", ctypes.c_uint64), ("pitch", ctypes.c_int64),
                ("scale_pitch", ctypes.c_int64), ("stride", ctypes.c_int64),
                ("scale_stride", ctypes.c_int64)]


class Adapters(ctypes.Structure):
    _fields_ = [*((n, ctypes.c_uint64) for n in ("down", "up", "scale", "order", "ends")),
                *((n, ctypes.c_int64) for n in ("down_pitch", "down_stride", "up_pitch",
                                                "up_stride")),
                ("factor", ctypes.c_float), ("count", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("format", ctypes.c_int32)]


class Sum(ctypes.Structure):
    _fields_ = [("z", ctypes.c_uint64), ("z_pitch", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("low", ctypes.c_uint64), ("largest", ctypes.c_uint64), ("out", ctypes.c_uint64),
                ("turned", ctypes.c_int64)]


A = 1 << 20  # an aligned address that nothing reads


def refused(rc, text):
    assert rc == BAD
    message = _native.load_library().srs_last_error().decode()
    assert text in message, message


def blocks(**changes):
    return ctypes.byref(Blocks(**{**dict(data=A, scale=A, rows=256, pitch=128, scale_pitch=1,
                                         format=3, square=1), **changes}))


def test_group_rows_refusals():
    call = _native.load_library().srs_group_rows
    for args, text in [
            ((A, 2, 8, 4, A, A), "4 or 8 bytes"), ((A, 4, 8, 0, A, A), "groups must be in"),
            ((A, 4, 8, 1025, A, A), "groups must be in"), ((A, 4, -1, 4, A, A), "rows must be in"),
            ((A, 4, 2**31, 4, A, A), "rows must be in"), ((None, 4, 8, 4, A, A), "null index"),
            ((A, 4, 8, 4, None, A), "null index"), ((A, 4, 8, 4, A, None), "null index"),
            ((A + 4, 8, 8, 4, A, A), "aligned"), ((A, 4, 8, 4, A + 2, A), "aligned")]:
        refused(call(*args, None), text)


def test_quantisation_refusals():
    lib = _native.load_library()
    copy = Copy(A, A, 128, 1, 128 * 64, 64)

    def stack(x=A, fmt=1, matrices=2, rows=64, cols=128, out=3, rule=0, to=copy):
        return lib.srs_quantize_stack(x, fmt, matrices, rows, cols, cols, rows * cols, out, rule, 1,
                                      0, 0, None if to is None else ctypes.byref(to), None, None)

    refused(stack(fmt=3), "input format")
    refused(stack(out=1), "output format")
    refused(stack(rule=9), "rounding rule")
    refused(stack(matrices=70000), "too large")
    refused(stack(matrices=-1), "negative")
    refused(stack(to=None), "null outputs")
    refused(stack(x=None), "null input")
    refused(stack(to=Copy(A, A, 64, 1, 128 * 64, 64)), "row length")
    refused(stack(to=Copy(A, A, 128, 1, 100, 64)), "16-byte")
    refused(stack(to=Copy(A, 0, 128, 1, 128 * 64, 64)), "no scale")
    refused(stack(cols=200, to=Copy(A, A, 208, 1, 208 * 64, 64)), "2 blocks a row")

    def groups(ends=A, n=4, turned=Copy(A, A, 1024, 32, 0, 0), rows=300):
        return lib.srs_quantize_groups(A, 1, rows, 64, 64, ends, n, 3, 0, 0, 0, None,
                                       None if turned is None else ctypes.byref(turned), None)

    refused(groups(ends=None), "ends")
    refused(groups(n=1025), "groups must be in")
    refused(groups(turned=None), "transposed copy")
    refused(groups(turned=Copy(A, A, 640, 32, 0, 0)), "row length")
    refused(groups(turned=Copy(A, A, 1024, 8, 0, 0)), "scale pitch")


def test_sizes_of_grouped_copies_hold_every_grouping():
    lib = _native.load_library()
    for rows, groups in ((1, 1), (1, 50), (127, 3), (128, 3), (300, 4), (5000, 64)):
        columns, scales = lib.srs_group_columns(rows, groups), lib.srs_group_scales(rows, groups)
        assert columns % 128 == 0 and scales % 4 == 0
        some = min(rows, groups)
        worst = [1] * (some - 1) + [rows - some + 1]  # as many groups with rows as there can be
        tiles = [-(-n // 128) for n in worst]
        assert columns >= 128 * sum(tiles) and scales >= sum(-(-t // 4) * 4 for t in tiles)
    assert lib.srs_group_columns(0, 4) == 0 == lib.srs_group_scales(0, 4)


def test_expert_refusals():
    lib = _native.load_library()

    def linear(w=None, experts=2, ends=A, rows=8, k=128, d=A, workspace=A, size=1 << 20, fmt=1):
        return lib.srs_expert_linear(A, fmt, rows, k, k, 3, w or blocks(), experts, ends, d,
                                     workspace, size, None)

    refused(linear(experts=0), "groups must be in")
    refused(linear(ends=None), "ends")
    refused(linear(experts=3), "not a multiple")
    refused(linear(w=blocks(format=1)), "unknown format")
    refused(linear(w=blocks(pitch=64)), "row pitch")
    refused(linear(w=blocks(rows=2**31)), "rows")
    refused(linear(d=None), "result pointer")
    refused(linear(d=A + 1), "result pointer")
    refused(linear(size=100), "workspace")
    refused(linear(workspace=None), "workspace")
    refused(linear(rows=-1), "negative")
    refused(lib.srs_expert_matmul(blocks(square=1), blocks(), 2, A, 128, A, 1, None), "1 x 128")
    refused(lib.srs_expert_matmul(blocks(square=0), blocks(), 2, A, 128, A, 5, None),
            "result format")
    turned = dict(square=0, pitch=1024, scale_pitch=32)
    gradient = lib.srs_expert_gradient
    refused(gradient(blocks(**turned), blocks(**{**turned, "square": 1}), 300, 4, A, A, 1, None),
            "transposed copy")
    refused(gradient(blocks(**turned), blocks(**{**turned, "scale_pitch": 8}), 300, 4, A, A, 1,
                     None), "transposed copy")
    refused(gradient(blocks(**turned), blocks(**turned), -1, 4, A, A, 1, None), "rows must be in")
    refused(gradient(blocks(**turned), blocks(**turned), 300, 4, A, None, 1, None),
            "result pointer")


def adapters(**changes):
    return ctypes.byref(Adapters(**{**dict(
        down=A, up=A, scale=0, order=A, ends=A, down_pitch=128, down_stride=128 * 8, up_pitch=8,
        up_stride=256 * 8, factor=1.0, count=3, rank=8, format=1), **changes}))


def test_adapter_refusals():
    lib = _native.load_library()

    def linear(a=None, tokens=100, k=128, pitch=128, x=A, w=None, fmt=3, rule=0, workspace=A,
               size=1 << 30):
        return lib.srs_adapter_linear(x, tokens, k, pitch, fmt, rule, 0, w or blocks(),
                                      a or adapters(), 0, A, None, None, workspace, size, None)

    for changes, text in [
            ({"count": 0}, "groups must be in"), ({"count": 1025}, "groups must be in"),
            ({"rank": 0}, "rank must be in"), ({"rank": 257}, "rank must be in"),
            ({"format": 0}, "BF16 or FP16"), ({"order": 0}, "order"), ({"ends": 0}, "ends"),
            ({"down": A + 8}, "16-byte"), ({"down_pitch": 100}, "16-byte"),
            ({"up": 0}, "16-byte"), ({"up_pitch": 4}, "16-byte"), ({"up_stride": 9}, "16-byte")]:
        refused(linear(a=adapters(**changes)), text)
    refused(linear(tokens=-1), "out of range")
    refused(linear(tokens=2**23), "out of range")
    refused(linear(x=A + 2), "16-byte")
    refused(linear(pitch=64), "16-byte")
    refused(linear(workspace=A + 16), "workspace")
    refused(linear(size=10), "workspace")

    def gradient(sums=1, fmt=1, tokens=100, rank=8, workspace=A, size=1 << 30, **changes):
        job = Sum(**{**dict(z=A, z_pitch=128, cols=128, low=A, largest=0, out=A, turned=0),
                     **changes})
        return lib.srs_adapter_gradient(ctypes.byref(job), sums, fmt, tokens, 3, rank, A, A,
                                        workspace, size, None)

    refused(gradient(sums=3), "one or two")
    refused(gradient(fmt=0), "BF16 or FP16")
    refused(gradient(rank=300), "out of range")
    refused(gradient(cols=-1), "out of range")
    refused(gradient(z=A + 8), "16-byte")
    refused(gradient(z_pitch=64), "16-byte")
    refused(gradient(out=0), "result pointer")
    refused(gradient(low=A + 8), "low needs a 16-byte")
    refused(gradient(low=0), "low needs a 16-byte")
    refused(gradient(largest=A + 2), "multiple of 4")
    refused(linear(a=adapters(scale=A + 2)), "scales")
    for low, largest in ((A + 2, None), (A, A + 1)):
        refused(lib.srs_adapter_linear(A, 100, 128, 128, 3, 0, 0, blocks(), adapters(), 0, A, low,
                                       largest, A, 1 << 30, None), "result pointer")


def test_struct_layouts():
    """The mirrors above against the header's own sizes, by what the compiler lays out."""
    assert ctypes.sizeof(Blocks) == 48 and ctypes.sizeof(Copy) == 48
    assert ctypes.sizeof(Adapters) == 88 and ctypes.sizeof(Sum) == 56


def test_python_refusals_without_a_gpu():
    x, w = torch.ones((4, 32)), torch.ones((2, 16, 32))
    with pytest.raises(ValueError, match="CUDA tensors"):
        sr_states.group_rows(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sr_states.expert_linear(x, w, torch.tensor([2, 4]))
    with pytest.raises(ValueError, match="CUDA tensors"):
        sr_states.quantize_stack(w)
    groups = sr_states.RowGroups(torch.zeros(4, dtype=torch.int32), torch.tensor([4]))
    down, up = torch.ones((1, 4, 32)), torch.ones((1, 16, 4))
    with pytest.raises(ValueError, match="CUDA tensors"):
        sr_states.adapter_linear(x, w[0], down, up, groups)
    with pytest.raises(TypeError, match="float8"):
        sr_states.expert_linear(x, w, torch.tensor([2, 4]), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sr_states.expert_linear(x, w, torch.tensor([2, 4]), grad_rounding="none")
    with pytest.raises(TypeError, match="pair of them"):
        sr_states.adapter_linear(x, (w[0], w[0]), down, up, groups)


def test_stacked_blocks_are_dequantised():
    scale = torch.tensor([[[127, 128]], [[126, 130]]], dtype=torch.uint8)
    data = torch.ones((2, 3, 200)).to(torch.float8_e4m3fn)
    held = sr_states.BlockTensor(data, scale.view(torch.float8_e8m0fnu)).dequantize()
    assert held.shape == (2, 3, 200)
    assert held[0, 0, 0] == 1 and held[0, 2, 199] == 2 and held[1, 1, 0] == 0.5
    assert held[1, 0, 128] == 8


def test_the_layers_draws_and_state():
    one = sr_states.BlockExperts(3, 8, 4, seed=7)
    assert one.weight.shape == (3, 4, 8) and (one.in_features, one.out_features) == (8, 4)
    x = torch.ones((2, 8), requires_grad=True)
    first, second = one._settings(x), one._settings(x)
    assert first["seed"] != second["seed"] and one.calls == 2
    other = sr_states.BlockExperts(3, 8, 4, seed=9)
    other.load_state_dict(one.state_dict())
    assert (other.seed, other.calls) == (7, 2) and torch.equal(other.weight, one.weight)
    assert other._settings(x) == one._settings(x)
    # layers made without a seed draw apart, linear and expert ones alike
    seeds = {sr_states.BlockExperts(2, 8, 4).seed, sr_states.BlockLinear(8, 4).seed,
             sr_states.BlockExperts(2, 8, 4).seed}
    assert len(seeds) == 3
