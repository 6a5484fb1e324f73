"""Muon, orthogonalize and FP8 blocks without a GPU: refusals that come before any
launch, the C ABI's own checks and its structure layouts."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import sr_states
from sr_states.cuda import _native

HEADER = Path(__file__).resolve().parents[1] / "include" / "srs_b200.h"


def newton(steps=5, eps=1e-7):
    h = _native.SrsNewton()
    h.steps, h.eps = steps, eps
    h.coefficients[:] = (3.4445, -4.775, 2.0315)
    return h


def test_cpu_tensors_are_refused():
    x = torch.ones(4, 128)
    for call in (lambda: sr_states.orthogonalize(x), lambda: sr_states.quantize_blocks(x),
                 lambda: sr_states.block_linear(x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    with pytest.raises(ValueError, match="CUDA"):
        sr_states.MuonSR([p]).step()


def test_muon_options_and_formats():
    p = torch.nn.Parameter(torch.ones(4, 4))
    opt = sr_states.MuonSR([p], state_dtype=torch.float8_e4m3fn)
    group = opt.param_groups[0]
    assert group["state_format"] == {"momentum_buffer": {"dtype": torch.float8_e4m3fn,
                                                         "rounding": "stochastic"}}
    assert sr_states.MuonRN([p]).param_groups[0]["state_format"]["momentum_buffer"]["rounding"] == (
        "nearest")
    again = sr_states.MuonSR([torch.nn.Parameter(torch.ones(4, 4))])
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["state_format"] == group["state_format"]
    for bad in ({"lr": -1}, {"momentum": 1.0}, {"weight_decay": -1}, {"scale": "x"},
                {"ns_steps": 0}, {"ns_coefficients": (1, 2)}, {"eps": -1}):
        with pytest.raises(ValueError):
            sr_states.MuonSR([p], **bad)
    with pytest.raises(ValueError, match="matrices"):
        sr_states.MuonSR([torch.nn.Parameter(torch.ones(4))])
    assert len(sr_states.MuonSR(iter([p])).param_groups[0]["params"]) == 1


def test_entry_points_check_before_any_cuda_call():
    lib, bad = _native.load_library(), _native.SRS_ERR_INVALID_ARGUMENT
    h = newton()
    orth = lambda **k: lib.srs_orthogonalize(*{  # noqa: E731
        "x": 256, "xf": 0, "rp": 8, "bs": 64, "y": 512, "yf": 0, "b": 1, "m": 8, "n": 8,
        "h": ctypes.byref(h), "w": 1024, "wb": 1 << 30, "s": None, **k}.values())
    assert orth(xf=3) == bad and b"format" in lib.srs_last_error()
    assert orth(m=-1) == bad and b"negative" in lib.srs_last_error()
    assert orth(m=1 << 25) == bad and b"large" in lib.srs_last_error()
    assert orth(h=ctypes.byref(newton(0))) == bad and b"steps" in lib.srs_last_error()
    assert orth(h=ctypes.byref(newton(eps=-1.0))) == bad and b"eps" in lib.srs_last_error()
    assert orth(x=None) == bad and orth(x=257) == bad
    assert orth(wb=16) == bad and b"workspace" in lib.srs_last_error()
    assert orth(w=1025) == bad
    assert orth(m=0) == _native.SRS_OK and orth(b=0) == _native.SRS_OK
    hp, rng = _native.SrsMuonHparams(), _native.SrsRng()

    def shapes(count=1, m=8, n=8):
        table = (_native.SrsMuonClass * 1)()
        table[0].count, table[0].m, table[0].n = count, m, n
        return table

    def matrix(param=256, grad=512, state=1024, flags=0):
        row = _native.SrsRow()
        row.param, row.grad, row.flags = param, grad, flags
        row.state[0] = state
        return ctypes.byref(row)

    rows = (_native.SrsRow * 1)()
    rows[0].param, rows[0].grad, rows[0].flags = 256, 512, 0
    rows[0].state[0] = 1024

    muon = lambda **k: lib.srs_muon_multi(*{  # noqa: E731
        "r": ctypes.byref(rows), "c": shapes(), "k": 1, "f": 1, "rule": 1, "hp": ctypes.byref(hp),
        "h": ctypes.byref(h), "rng": ctypes.byref(rng), "w": 1024, "wb": 1 << 30, "s": None,
        **k}.values())
    assert muon(f=9) == bad and muon(rule=9) == bad and muon(hp=None) == bad
    assert muon(r=None) == bad and muon(wb=0) == bad
    for r in (matrix(param=0), matrix(grad=0), matrix(state=0), matrix(param=258),
              matrix(grad=520, flags=_native.ROW_VECTOR_OK), matrix(state=1025)):
        assert muon(r=r) == bad, bytes(lib.srs_last_error())
    assert muon(c=None) == bad and muon(k=17) == bad and muon(k=-1) == bad
    for table in (shapes(count=0), shapes(m=0), shapes(n=-1), shapes(m=1 << 25), shapes(count=65)):
        assert muon(c=table) == bad and lib.srs_muon_workspace(table, 1) == -1
    assert lib.srs_muon_workspace(shapes(), 1) > 0 and lib.srs_muon_workspace(None, 0) == 0
    assert muon(k=0) == _native.SRS_OK
    quant = lambda **k: lib.srs_quantize_blocks(*{  # noqa: E731
        "x": 256, "xf": 0, "rows": 4, "cols": 64, "xp": 64, "of": 3, "rule": 0, "sq": 0,
        "seed": 0, "off": 0, "d": 512, "dp": 64, "s": 1024, "sp": 1, "dt": None, "dtp": 0,
        "st": None, "stp": 0, "stream": None, **k}.values())
    assert quant(of=1) == bad and quant(rule=7) == bad and quant(rows=-1) == bad
    assert quant(d=None) == bad and quant(d=520) == bad and quant(dp=72) == bad
    assert quant(dp=48) == bad and quant(s=None) == bad and quant(sp=0) == bad
    assert quant(x=None) == bad and quant(rows=0) == _native.SRS_OK

    def operand(**k):
        b = _native.SrsBlocks()
        for name, value in {"data": 256, "scale": 512, "rows": 4, "pitch": 128, "scale_pitch": 1,
                            "format": 3, "square": 0, **k}.items():
            setattr(b, name, value)
        return ctypes.byref(b)

    good = operand()
    mm = lib.srs_matmul_blocks
    for b in (operand(format=1), operand(rows=-1), operand(data=0), operand(data=264),
              operand(pitch=120), operand(pitch=64), operand(scale_pitch=0), None):
        assert mm(good, b, 128, 4096, 0, None) == bad
    assert mm(good, good, 128, None, 0, None) == bad and mm(good, good, -1, 4096, 0, None) == bad
    assert mm(good, good, 128, 4096, 4, None) == bad
    assert mm(operand(rows=0), good, 128, None, 0, None) == _native.SRS_OK
    need = lib.srs_linear_workspace(3, 100)
    assert need == 3 * (112 + 1) and lib.srs_linear_workspace(0, 5) == 0
    linear = lambda **k: lib.srs_linear_blocks(*{  # noqa: E731
        "x": 256, "xf": 0, "t": 3, "k": 100, "xp": 100, "bf": 3, "w": good, "d": 4096,
        "ws": 512, "wb": need, "s": None, **k}.values())
    assert linear(wb=need - 1) == bad and linear(ws=None) == bad and linear(ws=520) == bad
    assert linear(xf=5) == bad and linear(bf=1) == bad and linear(t=-1) == bad
    assert linear(w=None) == bad and linear(w=operand(pitch=96)) == bad and linear(x=None) == bad
    assert linear(t=0) == _native.SRS_OK
    assert lib.srs_copy_rows(256, 5, -1, 5, 512, 16, None) == bad
    assert lib.srs_copy_rows(256, 5, 1, 5, 520, 16, None) == bad
    assert lib.srs_copy_rows(256, 5, 1, 17, 512, 16, None) == bad
    assert lib.srs_copy_rows(None, 5, 1, 5, 512, 16, None) == bad
    assert lib.srs_copy_rows(None, 5, 0, 5, None, 16, None) == _native.SRS_OK


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_structure_layouts(tmp_path):
    probe = tmp_path / "layout.c"
    probe.write_text(f"""
#include <stddef.h>
#include <stdio.h>
#include "{HEADER}"
int main(void) {{
  printf("%zu %zu %zu %zu %zu %zu %d %zu %zu %d %d\\n", sizeof(srs_newton),
         offsetof(srs_newton, eps), sizeof(srs_muon_hparams), offsetof(srs_muon_hparams, nesterov),
         sizeof(srs_blocks), offsetof(srs_blocks, format), SRS_NEWTON_MAX_STEPS,
         sizeof(srs_muon_class), offsetof(srs_muon_class, neg_step), SRS_MUON_MAX_CLASSES,
         SRS_MUON_MAX_MATRICES);
  return 0;
}}
""")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", str(probe), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(_native.SrsNewton), _native.SrsNewton.eps.offset,
                   ctypes.sizeof(_native.SrsMuonHparams), _native.SrsMuonHparams.nesterov.offset,
                   ctypes.sizeof(_native.SrsBlocks), _native.SrsBlocks.format.offset,
                   _native.NEWTON_MAX_STEPS, ctypes.sizeof(_native.SrsMuonClass),
                   _native.SrsMuonClass.neg_step.offset, _native.MUON_MAX_CLASSES,
                   _native.MUON_MAX_MATRICES]
