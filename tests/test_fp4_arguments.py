"""CPU: arguments of the microscaled operators that contradict one another, and how sizes choose the few-rows kernel's launch."""
import ctypes
import os
import subprocess

import pytest
import torch

import int4linear_b200 as L
from conftest import ROOT
from int4linear_b200 import _lib, fp4


def test_quantize_refuses_a_format_that_is_not_its_outputs():
    cpu = torch.device("cpu")
    outs = {fmt: fp4.Fp4Matrix._new(4, 64, fmt, None, cpu) for fmt in fp4.FORMATS}
    for fmt, out in outs.items():
        assert fp4._wanted_format(None, out) == fmt and fp4._wanted_format(fmt, out) == fmt
        for other in [f for f in fp4.FORMATS if f != fmt] + ["fp4"]:
            with pytest.raises(ValueError):
                fp4._wanted_format(other, out)
    assert fp4._wanted_format(None, None) == "mxfp4" and fp4._wanted_format("nvfp4", None) == "nvfp4"


def test_few_rows_launches(tmp_path):
    exe = str(tmp_path / "fewrows_plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-o", exe,
                    os.path.join(ROOT, "tests", "fewrows_plan_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "FEWROWS_OK" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_quantize_into_an_output_of_another_format(cuda):
    x = torch.randn((4, 64), device=cuda)
    for fmt, other in (("mxfp4", "nvfp4"), ("nvfp4", "mxfp4")):
        out = L.quantize_fp4(x, fmt)
        codes = out.codes.clone()
        with pytest.raises(ValueError):
            L.quantize_fp4(-x, other, out=out)
        assert torch.equal(out.codes, codes)
        assert L.quantize_fp4(x, fmt, out=out) is out and L.quantize_fp4(x, out=out) is out
    assert L.quantize_fp4(x).format == "mxfp4"


def test_terms_of_the_gate_gradients():
    lib = _lib.load()
    one, two = 1 << 8, 1 << 9
    need = lib.int4_linear_fp4_grad_workspace_bytes
    m, n, k = 1030, 4100, 1056
    pitch = (n + 7) // 8 * 8
    piece = -(-m * pitch * 2 // 256) * 256
    assert need(m, n, k, 1 | one, 1, 1) == need(m, n, k, 1, 1, 1)                 # large: one term by itself
    assert need(m, n, k, 1 | two, 1, 1) == need(m, n, k, 1, 1, 1) + 2 * piece     # the second terms of dg and du
    assert need(64, 128, 128, 1 | two, 1, 1) == need(64, 128, 128, 1, 1, 1)       # small: two by itself
    assert need(64, 128, 128, 1 | one, 1, 1) < need(64, 128, 128, 1, 1, 1)
    assert need(m, n, k, 1 | one | two, 1, 1) == -1
    q = fp4._CMatrix(1 << 20, (1 << 20) + 4096, None, 8, 64, 0)
    for activation in (one | two, one | two | 1, one | 3):
        assert lib.int4_linear_fp4_gated_grad_async(*[1 << 20] * 3, *[ctypes.byref(q)] * 3, activation, *[1 << 20] * 4, 1 << 40, None) == 1
    assert lib.int4_linear_fp4_gated_launch_async(*[ctypes.byref(q)] * 3, two, 1 << 20, None, None, 0, None) == 1  # the backward's only
    for bad in (0, 3, "2"):
        with pytest.raises(ValueError):
            fp4._terms_flag(bad)


def test_workspace_of_sizes_that_no_call_takes():
    """Sizes beyond the operators' are refused before their bytes overflow."""
    need = _lib.load().int4_linear_fp4_grad_workspace_bytes
    for sizes in ((2 ** 31 - 1,) * 3, (2 ** 26 + 1, 8, 64), (8, 2 ** 26 + 1, 64), (8, 8, 2 ** 26 + 32)):
        for gated in (0, 1):
            assert need(*sizes, gated, 1, 1) == -7
    assert need(2 ** 26, 2 ** 26, 2 ** 26, 1, 1, 1) > 2 ** 54
