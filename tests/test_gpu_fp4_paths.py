"""GPU: forms of the microscaled backward passes by size, strided gradients, streams and threads.

Which form a size takes (operands expanded by a launch of their own or inside the products, dg and du in one or two terms,
contractions whole or cut) is checked on the CPU in test_fp4_plan.py for the same sizes."""
import threading

import pytest
import torch

import fp4_ref as R
import int4linear_b200 as L
from test_gpu_fp4 import close, grad_bounds

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp4", "nvfp4"]


def gated_reference(dh, gate, up, xv, gv, uv, act):
    """(want, bound) of dx, dwg and dwu where dg and du are rounded to bf16 once (as in test_gated_backward)."""
    g, u, d = gate.double(), up.double(), dh.double()
    dg, du = d * u * R.act_slope(g, act), d * R.act(g, act)
    soft = 2.0 ** -18 * (1 + g.abs()).clamp(max=9.0) * d.abs()
    eg, eu = dg.abs() * 2.0 ** -8 + soft * u.abs() * 1.01, du.abs() * 2.0 ** -8 + soft * 1.01
    out = []
    for pairs in (((dg, eg, gv), (du, eu, uv)), ((dg.t(), eg.t(), xv),), ((du.t(), eu.t(), xv),)):
        want = sum(a @ b for a, _, b in pairs)
        bound = sum(grad_bounds(a, b)[0] * len(pairs) * 1.01 + e @ b.abs() for a, e, b in pairs)
        out.append((want, (want.abs() + bound) * 2.0 ** -8 + bound))
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1030, 4096, 1056), (1030, 4101, 1056)])
def test_linear_backward_of_expanded_operands(cuda, fmt, m, n, k):
    x, w = R.matrix(L, m, k, fmt, m + k, cuda), R.matrix(L, n, k, fmt, n + k + 1, cuda, scale=2.0 ** -5)
    dy = torch.randn((m, n), device=cuda).to(torch.bfloat16)
    d, xv, wv = dy.double(), R.values(x), R.values(w)
    dx, dw = L.linear_fp4_backward(dy, x, w)
    for got, a, b in ((dx, d, wv), (dw, d.t(), xv)):
        want, acc = a @ b, grad_bounds(a, b)[0]
        close(got, want, (want.abs() + acc) * 2.0 ** -8 + acc)
    only_x, none = L.linear_fp4_backward(dy, x, w, need=(True, False))
    assert none is None and torch.equal(only_x, dx)
    none, only_w = L.linear_fp4_backward(dy, x, w, need=(False, True))
    assert none is None and torch.equal(only_w, dw)


# Operands expanded inside the products, dg and du in one term; the same with operands expanded first; contractions cut.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k,act", [(300, 4100, 1056, "silu"), (300, 4104, 1056, "gelu"), (512, 3000, 2080, "gelu_tanh"),
                                       (1030, 4100, 1056, "silu"), (515, 2731, 1056, "gelu_tanh")])
def test_gated_backward_in_one_term(cuda, fmt, m, n, k, act):
    x = R.matrix(L, m, k, fmt, m + k, cuda, scale=2.0 ** -2)
    wg, wu = R.matrix(L, n, k, fmt, n + k + 1, cuda, scale=2.0 ** -4), R.matrix(L, n, k, fmt, n + k + 2, cuda, scale=2.0 ** -3)
    gen = torch.Generator(device=cuda).manual_seed(m)
    dh, gate, up = ((torch.randn((m, n), generator=gen, device=cuda) * s).to(torch.bfloat16) for s in (1.0, 3.0, 2.0))
    grads = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act)
    for got, (want, bound) in zip(grads, gated_reference(dh, gate, up, R.values(x), R.values(wg), R.values(wu), act)):
        close(got, want, bound)
    only_x = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(True, False))[0]
    only_w = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(False, True))[1:]
    for got, want in zip((only_x, *only_w), grads):
        assert torch.equal(got, want)
    for _ in range(4):  # nothing depends on timing
        for got, want in zip(L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act), grads):
            assert torch.equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k,act", [(300, 4100, 1056, "silu"), (1030, 4100, 1056, "gelu"), (515, 2731, 1056, "gelu_tanh"), (90, 200, 128, "silu")])
def test_terms_decide_the_rounding(cuda, fmt, m, n, k, act):
    """Two terms: an error of 2^-16 in dg and du, so what is left is the result's rounding.  One: another 2^-9 in the mean square.
    Where the sizes decide, the bits are those of one or the other."""
    x, wg, wu = (R.matrix(L, r, k, fmt, i, cuda, scale=0.25) for i, r in enumerate((m, n, n)))
    gen = torch.Generator(device=cuda).manual_seed(m)
    dh, gate, up = (torch.randn((m, n), generator=gen, device=cuda).to(torch.bfloat16) for _ in range(3))
    g, u, d = gate.double(), up.double(), dh.double()
    dg, du = d * u * R.act_slope(g, act), d * R.act(g, act)
    xv, gv, uv = R.values(x), R.values(wg), R.values(wu)
    want = (dg @ gv + du @ uv, dg.t() @ xv, du.t() @ xv)
    one, two, auto = (L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, terms=t) for t in (1, 2, None))
    for a, b, w in zip(one, two, want):
        rounding = (w.to(torch.bfloat16).double() - w).norm()
        assert (b.double() - w).norm() <= 1.05 * rounding < (a.double() - w).norm() <= 2 * rounding
    for a, b in zip(auto, two if m * n <= 65536 else one):
        assert torch.equal(a, b)
    only_x = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(True, False), terms=2)[0]
    only_w = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(False, True), terms=2)[1:]
    for a, b in zip((only_x, *only_w), two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m,n", [(70, 264), (70, 131), (700, 1000)])
def test_strided_gradients(cuda, m, n):
    x, wg, wu = (R.matrix(L, r, 96, "nvfp4", i, cuda) for i, r in enumerate((m, n, n)))
    wide = torch.randn((3, m, 2 * n + 5), device=cuda).to(torch.bfloat16)
    rows = [t[:, 3:n + 3] for t in wide]
    every = [t[:, 1:2 * n + 1:2] for t in wide]
    turned = [t[:, :n].t().contiguous().t() for t in wide]
    spread = [t[:1, :n].expand(m, n) for t in wide]
    for views in (rows, every, turned, spread):
        copies = [t.contiguous() for t in views]
        for a, b in zip(L.gated_linear_fp4_backward(*views, x, wg, wu, "gelu"), L.gated_linear_fp4_backward(*copies, x, wg, wu, "gelu")):
            assert torch.equal(a, b)
        for a, b in zip(L.linear_fp4_backward(views[0], x, wg), L.linear_fp4_backward(copies[0], x, wg)):
            assert torch.equal(a, b)


def every_operator(x, wg, wu, wd, dy, fmt, stream=None):
    """A training step of a feed-forward block with every operator in it."""
    xq = L.quantize_fp4(x, fmt, stream=stream)
    h, g, u = L.gated_linear_fp4(xq, wg, wu, "gelu", save=True, stream=stream)
    hq = L.quantize_fp4(h, fmt, stream=stream)
    y = L.linear_fp4(hq, wd, stream=stream)
    dh, dwd = L.linear_fp4_backward(dy, hq, wd, stream=stream)
    grads = L.gated_linear_fp4_backward(dh, g, u, xq, wg, wu, "gelu", stream=stream)
    return (L.dequantize_fp4(xq, stream=stream), L.dequantize_fp4(hq, dtype=torch.float16, stream=stream), h, g, u, y, dh, dwd, *grads)


def block_operands(m, k, n, fmt, seed, device):
    gen = torch.Generator(device=device).manual_seed(seed)
    x, dy = (torch.randn((m, k), generator=gen, device=device).to(torch.bfloat16) for _ in range(2))
    return (x, *(R.matrix(L, r, c, fmt, seed + i, device, scale=2.0 ** -4) for i, (r, c) in enumerate(((n, k), (n, k), (k, n)))), dy, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_operator_on_another_stream(cuda, fmt):
    ops = block_operands(150, 512, 1376, fmt, 1, cuda)
    want = every_operator(*ops)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream, torch.cuda.current_stream(), torch.cuda.default_stream()):
        got = every_operator(*ops, stream=stream)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    with torch.cuda.stream(side):
        got = every_operator(*ops)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert L.last_status() == 0


def test_threads_share_the_device(cuda):
    """Several host threads, each with operands and a stream of its own, all operators at once."""
    work = [(block_operands(m, 256, 608, fmt, 10 * i + 1, cuda)) for i, (m, fmt) in enumerate(((3, "mxfp4"), (40, "nvfp4"), (130, "mxfp4"), (300, "nvfp4")))]
    want = [every_operator(*ops) for ops in work]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = every_operator(*work[i])
                    stream.synchronize()
                    for a, b in zip(got, want[i]):
                        if not torch.equal(a, b):
                            raise AssertionError(f"thread {i} differs")
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert L.last_status() == 0
