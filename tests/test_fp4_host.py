"""CPU: argument checks of the microscaled 4-bit operators, the reference they are tested against, and the schedule
of the backward pass (no GPU needed)."""
import copy
import ctypes
import os
import pickle
import subprocess

import pytest
import torch

import fp4_ref as R
import int4linear_b200 as L
import int4linear_b200.torch_op  # noqa: F401  (registers torch.ops.int4linear.*)
from conftest import ROOT
from int4linear_b200 import _lib, fp4

BASE = 1 << 20  # a device address that nothing looks at before the checks


def matrix(rows=8, k=64, fmt=0, codes=BASE, scales=BASE + 4096, ts=None):
    return fp4._CMatrix(codes, scales, ts, rows, k, fmt)


def bad_matrices():
    """(matrix, status) pairs that every entry point refuses."""
    return [(matrix(rows=0), 1), (matrix(rows=-1), 1), (matrix(k=0), 1), (matrix(k=48), 2), (matrix(k=16), 2), (matrix(fmt=2), 1), (matrix(fmt=-1), 1),
            (matrix(codes=None), 1), (matrix(scales=None), 1), (matrix(codes=BASE + 8), 3), (matrix(scales=BASE + 4), 3),
            (matrix(ts=BASE), 1), (matrix(fmt=1, ts=BASE + 2), 3), (matrix(rows=2 ** 26 + 1), 7), (matrix(k=2 ** 26 + 32), 7)]


def test_c_entry_points_refuse_bad_matrices():
    lib = _lib.load()
    ok = matrix()
    ref = ctypes.byref
    big = 1 << 40
    for q, status in bad_matrices() + [(None, 1)]:
        p = ref(q) if q is not None else None
        assert lib.int4_linear_fp4_quantize_async(BASE, 0, 64, p, None) == status
        assert lib.int4_linear_fp4_dequantize_async(p, BASE, 0, None) == status
        for x, w in ((p, ref(ok)), (ref(ok), p)):
            assert lib.int4_linear_fp4_launch_async(x, w, None, BASE, 0, None) == status
            assert lib.int4_linear_fp4_grad_async(BASE, x, w, BASE, BASE, BASE, big, None) == status
            assert lib.int4_linear_fp4_gated_launch_async(x, w, ref(ok), 0, BASE, None, None, 0, None) == status
            assert lib.int4_linear_fp4_gated_grad_async(BASE, BASE, BASE, x, w, ref(ok), 0, BASE, BASE, BASE, BASE, big, None) == status
        assert lib.int4_linear_fp4_gated_launch_async(ref(ok), ref(ok), p, 0, BASE, None, None, 0, None) == status
        assert lib.int4_linear_last_status() == status


def test_c_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    ref = ctypes.byref
    ok, wide, nv, tall = matrix(), matrix(k=96), matrix(fmt=1), matrix(rows=9)
    big = 1 << 40
    q = lib.int4_linear_fp4_quantize_async
    assert q(None, 0, 64, ref(ok), None) == 1
    assert q(BASE, 3, 64, ref(ok), None) == 1 and q(BASE, -1, 64, ref(ok), None) == 1
    assert q(BASE, 0, 63, ref(ok), None) == 1  # rows overlap
    assert q(BASE + 1, 0, 64, ref(ok), None) == 3 and q(BASE + 2, 2, 64, ref(ok), None) == 3
    d = lib.int4_linear_fp4_dequantize_async
    assert d(ref(ok), None, 0, None) == 1 and d(ref(ok), BASE, 3, None) == 1 and d(ref(ok), BASE + 8, 0, None) == 3
    y = lib.int4_linear_fp4_launch_async
    assert y(ref(ok), ref(wide), None, BASE, 0, None) == 1   # k differs
    assert y(ref(ok), ref(nv), None, BASE, 0, None) == 1     # format differs
    assert y(ref(ok), ref(ok), None, None, 0, None) == 1
    assert y(ref(ok), ref(ok), None, BASE, 2, None) == 1     # fp32 output
    assert y(ref(ok), ref(ok), BASE + 2, BASE, 0, None) == 3
    assert y(ref(ok), ref(ok), None, BASE + 8, 0, None) == 3
    g = lib.int4_linear_fp4_gated_launch_async
    assert g(ref(ok), ref(ok), ref(tall), 0, BASE, None, None, 0, None) == 1   # weights differ in rows
    assert g(ref(ok), ref(ok), ref(ok), 3, BASE, None, None, 0, None) == 1
    assert g(ref(ok), ref(ok), ref(ok), 0, BASE, BASE, None, 0, None) == 1     # gate without up
    assert g(ref(ok), ref(ok), ref(ok), 0, BASE, BASE + 2, BASE, 0, None) == 3
    b = lib.int4_linear_fp4_grad_async
    assert lib.int4_linear_fp4_grad_workspace_bytes(8, 8, 64, 0, 1, 1) == 0  # nothing to lay out anew
    odd = matrix(rows=9)
    need = lib.int4_linear_fp4_grad_workspace_bytes(8, 9, 64, 0, 1, 1)
    assert need > 0 and need % 256 == 0
    assert b(None, ref(ok), ref(ok), BASE, BASE, BASE, need, None) == 1
    assert b(BASE, ref(ok), ref(ok), None, None, BASE, need, None) == 1       # nothing wanted
    assert b(BASE, ref(ok), ref(odd), BASE, BASE, BASE, need - 1, None) == 1  # workspace too small
    assert b(BASE, ref(ok), ref(odd), BASE, BASE, None, need, None) == 1
    assert b(BASE, ref(ok), ref(ok), BASE, BASE, BASE + 128, big, None) == 3
    assert b(BASE + 2, ref(ok), ref(ok), BASE, BASE, BASE, need, None) == 3   # n % 8 == 0: 16-byte rows
    h = lib.int4_linear_fp4_gated_grad_async
    assert h(BASE, None, BASE, ref(ok), ref(ok), ref(ok), 0, BASE, BASE, BASE, BASE, big, None) == 1
    assert h(BASE, BASE, BASE, ref(ok), ref(ok), ref(ok), 0, BASE, BASE, None, BASE, big, None) == 1  # one weight gradient
    assert h(BASE, BASE, BASE, ref(ok), ref(ok), ref(ok), 7, BASE, BASE, BASE, BASE, big, None) == 1
    assert lib.int4_linear_fp4_grad_workspace_bytes(0, 8, 64, 0, 1, 1) == -1
    assert lib.int4_linear_fp4_grad_workspace_bytes(4096, 14336, 4096, 1, 1, 1) >= 2 * (2 * 4096 * 14336 + 2 * 14336 * 4096 + 4096 * 4096)


def test_no_gpu_means_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib = _lib.load()
    ok = ctypes.byref(matrix())
    assert lib.int4_linear_fp4_quantize_async(BASE, 0, 64, ok, None) == 6
    assert lib.int4_linear_fp4_launch_async(ok, ok, None, BASE, 0, None) == 6


def test_scale_bytes():
    lib = _lib.load()
    for rows, k, fmt in ((1, 32, "mxfp4"), (128, 128, "mxfp4"), (129, 160, "mxfp4"), (1, 32, "nvfp4"), (300, 4096, "nvfp4")):
        assert lib.int4_linear_fp4_scale_bytes(rows, k, fp4.FORMATS[fmt]) == fp4._scale_bytes(rows, k, fmt)
    assert fp4._scale_bytes(129, 160, "mxfp4") == 2 * 2 * 512 and fp4._scale_bytes(1, 32, "nvfp4") == 512
    for bad in ((0, 32, 0), (1, 48, 0), (1, 32, 2)):
        assert lib.int4_linear_fp4_scale_bytes(*bad) == -1


def test_python_refuses_cpu_tensors_and_unknown_names():
    x = torch.zeros((4, 64))
    with pytest.raises(ValueError):
        L.quantize_fp4(x)
    with pytest.raises(ValueError):
        L.Fp4Matrix(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 4, 64)
    with pytest.raises(ValueError):
        fp4._check_shape(4, 64, "fp4")
    for rows, k in ((4, 48), (4, 0), (-1, 32), (2 ** 26 + 1, 32), (1, 2 ** 26 + 32)):
        with pytest.raises(ValueError):
            fp4._check_shape(rows, k, "mxfp4")
    with pytest.raises(ValueError):
        fp4._check_act("relu")
    with pytest.raises(ValueError):
        fp4._half(torch.float32, None)
    with pytest.raises(TypeError):
        fp4._type_of(torch.float64)
    with pytest.raises(ValueError):
        fp4._check_tensor_scale(torch.ones(1), "mxfp4", torch.device("cpu"))
    with pytest.raises(ValueError):
        fp4._check_tensor_scale(torch.ones(2), "nvfp4", torch.device("cpu"))


def test_ops_are_registered_with_shape_inference():
    x = torch.empty((5, 64), device="meta", dtype=torch.bfloat16)
    c, s = torch.ops.int4linear.quantize_fp4(x, "nvfp4", None)
    assert c.shape == (5, 32) and c.dtype == torch.uint8 and s.shape == (512,)
    wc, ws = torch.ops.int4linear.quantize_fp4(torch.empty((9, 64), device="meta"), "nvfp4", None)
    y = torch.ops.int4linear.linear_fp4(c, s, None, wc, ws, None, None, "nvfp4")
    assert y.shape == (5, 9) and y.dtype == torch.bfloat16
    h = torch.ops.int4linear.gated_linear_fp4(c, s, None, wc, ws, None, wc, ws, None, "silu", "nvfp4")
    assert h.shape == (5, 9) and h.dtype == torch.bfloat16
    with pytest.raises(Exception):
        torch.ops.int4linear.linear_fp4(c, s, None, wc[:, :16], ws, None, None, "nvfp4")
    with pytest.raises(Exception):
        torch.ops.int4linear.quantize_fp4(x[:, :40], "nvfp4", None)


def test_reference_quantiser_by_brute_force():
    """The reference itself: every e2m1 and e4m3 value maps to itself, borders go to the even code, and the chosen
    code and scale are never farther from the value than any other."""
    mag = torch.tensor(R.MAG, dtype=torch.float64)
    grid = R.e4m3_values()
    assert torch.equal(grid.float(), torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float())
    for g in (mag, grid):
        assert torch.equal(R.nearest_even(g, g), torch.arange(g.numel()))
        mid = (g[1:] + g[:-1]) / 2
        idx = R.nearest_even(mid, g)
        assert (idx % 2 == 0).all()
        v = torch.rand(5000, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * g[-1]
        assert torch.equal((v - g[R.nearest_even(v, g)]).abs(), (v[:, None] - g).abs().amin(1))
    x = torch.randn((64, 96), generator=torch.Generator().manual_seed(1))
    for fmt in ("mxfp4", "nvfp4"):
        codes, sb, finite = R.quantize(x, fmt)
        assert finite.all() and codes.shape == (64, 48)
        amax = x.view(64, -1, R.BLOCK[fmt]).abs().amax(-1).double()
        s = R.scale_values(sb, fmt)
        if fmt == "mxfp4":
            assert ((amax / s >= 4) & (amax / s < 8)).all()
        else:
            assert ((amax / 6 - s).abs() <= s / 16).all()


def test_reference_gradients_are_the_derivative():
    """The formulas the backward tests use, against central differences."""
    g = torch.linspace(-6, 6, 101, dtype=torch.float64)
    for kind in ("silu", "gelu", "gelu_tanh"):
        t = 1e-6
        diff = (R.act(g + t, kind) - R.act(g - t, kind)) / (2 * t)
        assert (R.act_slope(g, kind) - diff).abs().max() < 1e-8


def test_backward_tiles_are_dealt_out_once(tmp_path):
    exe = str(tmp_path / "grad_schedule_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "grad_schedule_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "DEAL_OK" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_copies_and_ops_on_the_gpu(cuda):
    x = torch.randn((5, 96), device=cuda)
    w = torch.randn((7, 96), device=cuda).to(torch.bfloat16)
    ts = torch.tensor([0.01], device=cuda)
    xq, wq = L.quantize_fp4(x, "nvfp4", tensor_scale=ts), L.quantize_fp4(w, "nvfp4")
    want = L.linear_fp4(xq, wq)
    for q in (copy.copy(xq), copy.deepcopy(xq), pickle.loads(pickle.dumps(xq))):
        assert torch.equal(L.linear_fp4(q, wq), want) and q.shape == (5, 96)
    c, s = torch.ops.int4linear.quantize_fp4(x, "nvfp4", ts)
    assert torch.equal(c, xq.codes) and torch.equal(s, xq.scales)
    assert torch.equal(torch.ops.int4linear.linear_fp4(c, s, ts, wq.codes, wq.scales, None, None, "nvfp4"), want)
    h = torch.ops.int4linear.gated_linear_fp4(c, s, ts, wq.codes, wq.scales, None, wq.codes, wq.scales, None, "gelu", "nvfp4")
    assert torch.equal(h, L.gated_linear_fp4(xq, wq, wq, "gelu"))


@pytest.mark.gpu
def test_python_refusals_on_the_gpu(cuda):
    x = torch.randn((5, 64), device=cuda)
    q, v, w = L.quantize_fp4(x), L.quantize_fp4(x, "nvfp4"), L.quantize_fp4(torch.randn((6, 96), device=cuda))
    with pytest.raises(TypeError):
        L.quantize_fp4(x.double())
    for bad in (x[0], x[:, :48]):
        with pytest.raises(ValueError):
            L.quantize_fp4(bad)
    with pytest.raises(ValueError):
        L.quantize_fp4(x, out=w)
    with pytest.raises(ValueError):
        L.quantize_fp4(x, "mxfp4", tensor_scale=torch.ones(1, device=cuda))
    for a, b in ((q, v), (q, w)):
        with pytest.raises(ValueError):
            L.linear_fp4(a, b)
        with pytest.raises(ValueError):
            L.gated_linear_fp4(a, a, b)
    y = torch.empty((5, 5), dtype=torch.bfloat16, device=cuda)
    for out in (y.t()[:, :4], y.float(), torch.empty((5, 6), dtype=torch.bfloat16, device=cuda)):
        with pytest.raises(ValueError):
            L.linear_fp4(q, q, out=out)
    with pytest.raises(ValueError):
        L.linear_fp4(q, q, out=y, dtype=torch.float16)
    with pytest.raises(L.Int4LinearError):  # not on a 16-byte boundary
        L.linear_fp4(q, q, out=torch.empty(26, dtype=torch.bfloat16, device=cuda)[1:].view(5, 5))
    for bias in (torch.ones(5, device=cuda, dtype=torch.bfloat16), torch.ones(6, device=cuda), torch.ones(5)):
        with pytest.raises(ValueError):
            L.linear_fp4(q, q, bias=bias)
    for dy in (y.float(), y[:4], y.to(torch.float16)):
        with pytest.raises(ValueError):
            L.linear_fp4_backward(dy, q, q)
        with pytest.raises(ValueError):
            L.gated_linear_fp4_backward(y, dy, y, q, q, q)
    with pytest.raises(ValueError):
        L.Fp4Matrix(q.codes, q.scales[:-1], 5, 64)
    with pytest.raises(ValueError):
        L.Fp4Matrix(q.codes, q.scales, 5, 96)
    assert L.linear_fp4_backward(y, q, q, need=(False, False)) == (None, None)
