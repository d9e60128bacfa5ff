"""GPU: microscaled 4-bit floating point against 64-bit references.

Tolerances.  Quantisation and expansion to fp32 are exact.  A product's error is bounded by one half step of the
output type (eps / 2, relative) plus the accumulation bound of fp4_ref.product_bound; a gated product's by the
same bounds carried through h = act(g) u with |act'| <= 1.13; a gradient's additionally by the rounding of the
incoming gradient to bf16 (2^-8 of every term)."""
import pytest
import torch

import fp4_ref as R
import int4linear_b200 as L

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp4", "nvfp4"]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def close(got, want, bound):
    got = got.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"worst excess {worst}, at error {err.max().item()}"


def ts_tensor(v, device):
    return torch.tensor([v], dtype=torch.float32, device=device)


# ---------------------------------------------------------------------------------------- quantisation

def check_quantized(x, fmt, ts, q):
    codes, sb, finite = R.quantize(x, fmt, ts)
    assert torch.equal(q.scale_rows(), sb)
    block = R.BLOCK[fmt]
    same = (q.codes == codes).view(x.shape[0], -1, block // 2)
    assert same[finite].all()
    # Padding of the scale tiles: zeros.
    full = q.scales.view(-(-x.shape[0] // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-x.shape[0] // 128) * 128, -1)
    assert not full[x.shape[0]:].any() and not full[:, sb.shape[1]:].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (16, 4096), (130, 96), (257, 1056), (1000, 288)])
def test_quantize_matches_definition(cuda, fmt, dtype, rows, k):
    gen = torch.Generator(device=cuda).manual_seed(rows * 1000 + k)
    x = (torch.randn((rows, k), generator=gen, device=cuda) * torch.exp(2 * torch.randn((rows, 1), generator=gen, device=cuda))).to(dtype)
    ts = ts_tensor(0.013, cuda) if fmt == "nvfp4" else None
    check_quantized(x, fmt, ts, L.quantize_fp4(x, fmt, tensor_scale=ts))
    check_quantized(x, fmt, None, L.quantize_fp4(x, fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_every_border(cuda, fmt):
    """Each tie between two codes and its two fp32 neighbours, under scales with every mantissa."""
    block = R.BLOCK[fmt]
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in (R.e4m3_values()[1:].float() if fmt == "nvfp4" else torch.exp2(torch.arange(-126.0, 125.0))):
        base = ties * s
        v = torch.cat((torch.nextafter(base, torch.zeros(())), base, torch.nextafter(base, torch.full((), torch.inf))))
        for signed in (v, -v):
            for part in signed.split(block - 1):
                row = torch.zeros(block)
                row[:part.numel()] = part
                row[block - 1] = 6.0 * s  # pins the scale: 6 s / 6, and the binade [4, 8) of a power of two
                rows.append(row)
    x = torch.stack(rows)
    x = torch.nn.functional.pad(x, (0, 32 - block)).to(cuda) if block < 32 else x.to(cuda)
    check_quantized(x, fmt, None, L.quantize_fp4(x, fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_scale_borders_and_specials(cuda, fmt):
    block = R.BLOCK[fmt]
    tops = [0.0, -0.0, 2.0 ** -149, 2.0 ** -127, 2.0 ** -126, 1.0, 3.9999998, 4.0, 7.9999995, 8.0, 2.0 ** 120, 3.4028235e38]
    grid = R.e4m3_values().float()
    for mid in ((grid[1:] + grid[:-1]) / 2 * 6).tolist():  # ties between two e4m3 scales
        m = torch.tensor(mid)
        tops += [float(torch.nextafter(m, torch.tensor(0.0))), mid, float(torch.nextafter(m, torch.tensor(1e9)))]
    tops += [448.0 * 6, 448.0 * 6 * 1.2, 1e6]
    x = torch.zeros((len(tops), 64))
    gen = torch.Generator().manual_seed(3)
    x[:, :block] = torch.rand((len(tops), block), generator=gen) * torch.tensor(tops).unsqueeze(1)
    x[:, 1] = torch.tensor(tops)
    x[:, block:] = torch.randn((len(tops), 64 - block), generator=gen)
    x = x.to(cuda)
    check_quantized(x, fmt, None, L.quantize_fp4(x, fmt))
    bad = torch.randn((6, 96), generator=gen)
    bad[1, 5], bad[2, 40], bad[3, 95], bad[4, 0] = float("inf"), float("nan"), float("-inf"), float("nan")
    bad = bad.to(cuda)
    q = L.quantize_fp4(bad, fmt)
    check_quantized(bad, fmt, None, q)
    v = L.dequantize_fp4(q)
    blocks = torch.isnan(v).view(6, -1, block)
    assert torch.equal(blocks.all(-1), blocks.any(-1)) and int(blocks.all(-1).sum()) == 4


def test_quantize_tensor_scale_zero_and_saturation(cuda):
    x = torch.randn((5, 64), device=cuda)
    q = L.quantize_fp4(x, "nvfp4", tensor_scale=ts_tensor(0.0, cuda))
    assert not (q.codes & 0x77).any() and not q.scales.any()
    assert not L.dequantize_fp4(q).any()
    q = L.quantize_fp4(x * 1e6, "nvfp4", tensor_scale=ts_tensor(1.0, cuda))  # far beyond 448 * 6
    assert L.dequantize_fp4(q).abs().max().item() == 448.0 * 6


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_strided_and_unaligned(cuda, fmt):
    big = torch.randn((70, 515), device=cuda, dtype=torch.bfloat16)
    for view in (big[:, :96], big[:, 3:163], big[::2, 8:40], big[5:6, 1:65], big.t()[:512].t()[:, :512], big[:, :128].t()[:96, :64],
                 big[:1, :64].expand(9, 64)):
        want = L.quantize_fp4(view.contiguous(), fmt)
        got = L.quantize_fp4(view, fmt)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_into_out_leaves_the_rest(cuda, fmt):
    x = torch.randn((5, 96), device=cuda)
    want = L.quantize_fp4(x, fmt)
    pool = torch.full((5 * 48 + 64,), 0xAB, dtype=torch.uint8, device=cuda)
    spool = torch.full((want.scales.numel() + 64,), 0xCD, dtype=torch.uint8, device=cuda)
    out = L.Fp4Matrix(pool[32:32 + 240].view(5, 48), spool[16:16 + want.scales.numel()], 5, 96, fmt)
    assert L.quantize_fp4(x, out=out) is out
    assert torch.equal(out.codes, want.codes) and torch.equal(out.scales, want.scales)
    assert (pool[:32] == 0xAB).all() and (pool[272:] == 0xAB).all() and (spool[:16] == 0xCD).all() and (spool[16 + want.scales.numel():] == 0xCD).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k", [(1, 32), (129, 160), (300, 2048)])
def test_dequantize(cuda, fmt, rows, k):
    q = R.matrix(L, rows, k, fmt, rows + k, cuda, scale=2.0 ** -4)
    want = R.values(q)
    got = L.dequantize_fp4(q)
    close(got, want, want.abs() * 2.0 ** -24)
    for dtype, half in HALF.items():
        close(L.dequantize_fp4(q, dtype=dtype), want, want.abs() * (half + 2.0 ** -24) + TINY[dtype])


def test_dequantize_every_scale_byte(cuda):
    for fmt in FORMATS:
        n = 256 if fmt == "mxfp4" else 128
        codes = torch.arange(16, dtype=torch.uint8).repeat(n, R.BLOCK[fmt] // 16 * 2)[:, :32]
        packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
        sb = torch.arange(n, dtype=torch.uint8).view(n, 1).repeat(1, 32 // R.BLOCK[fmt])
        q = L.Fp4Matrix.from_rows(packed.to(cuda), sb.to(cuda), fmt)
        got, want = L.dequantize_fp4(q).double(), R.values(q)
        # 2^128 = 2 * 2^127 already lies beyond the largest float, 2^128 (1 - 2^-24)
        want = torch.where(want.abs() >= 2.0 ** 128, torch.copysign(torch.full_like(want, torch.inf), want), want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


def test_scale_order_round_trip(cuda):
    for fmt in FORMATS:
        q = R.matrix(L, 300, 352, fmt, 9, cuda)
        again = L.Fp4Matrix.from_rows(q.codes, q.scale_rows(), fmt, q.tensor_scale)
        assert torch.equal(again.scales, q.scales)


# ---------------------------------------------------------------------------------------------- product

SHAPES = [(1, 1, 32), (1, 128, 256), (2, 40, 64), (16, 14336 // 16, 4096), (5, 250, 992), (31, 64, 96), (33, 129, 160),
          (64, 1000, 512), (100, 77, 288), (128, 256, 256), (129, 257, 1056), (200, 512, 2080), (257, 385, 544),
          (300, 1024, 8192), (513, 520, 32), (65, 200, 6400), (129, 1000, 8192), (256, 130, 14336)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(cuda, fmt, m, n, k):
    x, w = R.matrix(L, m, k, fmt, m + k, cuda), R.matrix(L, n, k, fmt, n + k + 1, cuda, scale=2.0 ** -5)
    xv, wv = R.values(x), R.values(w)
    want, acc = xv @ wv.t(), R.product_bound(xv, wv)
    for dtype, half in HALF.items():
        close(L.linear_fp4(x, w, dtype=dtype), want, want.abs() * half + acc * (1 + half) + TINY[dtype])
    bias = torch.randn((n,), device=cuda)
    want = want + bias.double()
    close(L.linear_fp4(x, w, bias=bias), want, want.abs() * 2.0 ** -8 + (acc + 2.0 ** -23 * (want.abs() + bias.abs().double())) * 1.01)


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_many_tiles(cuda, fmt):
    """More tiles than the GPU holds at once: every worker computes several, accumulators alternate."""
    m, n, k = 1500, 7000, 288
    x, w = R.matrix(L, m, k, fmt, 1, cuda), R.matrix(L, n, k, fmt, 2, cuda, scale=2.0 ** -5)
    xv, wv = R.values(x), R.values(w)
    want = xv @ wv.t()
    close(L.linear_fp4(x, w), want, want.abs() * 2.0 ** -8 + R.product_bound(xv, wv) * 1.01)
    n = 7001
    w = R.matrix(L, n, k, fmt, 3, cuda, scale=2.0 ** -5)
    want = xv @ R.values(w).t()
    close(L.linear_fp4(x, w), want, want.abs() * 2.0 ** -8 + R.product_bound(xv, R.values(w)) * 1.01)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 300])
def test_linear_exact_integers(cuda, fmt, m):
    """Integer-valued operands: every partial sum is exact, so is the result (below 2^8 in bf16)."""
    gen = torch.Generator().manual_seed(m)
    n, k = 270, 320
    xi = torch.zeros((m, k), dtype=torch.uint8)
    wi = torch.zeros((n, k), dtype=torch.uint8)
    for t in (xi, wi):
        t[:, ::4] = torch.tensor([2, 10, 0], dtype=torch.uint8)[torch.randint(0, 3, t[:, ::4].shape, generator=gen)]  # 1, -1, 0
    one = 127 if fmt == "mxfp4" else 0x38
    mats = [L.Fp4Matrix.from_rows((t[:, 0::2] | (t[:, 1::2] << 4)).to(cuda),
                                  torch.full((t.shape[0], k // R.BLOCK[fmt]), one, dtype=torch.uint8, device=cuda), fmt) for t in (xi, wi)]
    want = R.values(mats[0]) @ R.values(mats[1]).t()
    assert want.abs().max() <= 80
    assert torch.equal(L.linear_fp4(*mats).double(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [2, 20, 260])
def test_linear_nan_stays_in_its_row_and_column(cuda, fmt, m):
    n, k = 140, 416
    x, w = R.matrix(L, m, k, fmt, 5, cuda), R.matrix(L, n, k, fmt, 6, cuda)
    clean = L.linear_fp4(x, w)
    sx, sw = x.scale_rows(), w.scale_rows()
    nan = 255 if fmt == "mxfp4" else 0x7F
    sx[1, -1], sw[77, 0] = nan, nan
    y = L.linear_fp4(L.Fp4Matrix.from_rows(x.codes, sx, fmt, x.tensor_scale), L.Fp4Matrix.from_rows(w.codes, sw, fmt, w.tensor_scale))
    hit = torch.zeros((m, n), dtype=torch.bool, device=cuda)
    hit[1], hit[:, 77] = True, True
    assert torch.isnan(y[hit]).all()
    assert torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("m,n", [(7, 200), (150, 200), (150, 201), (7, 201)])
def test_linear_out_view_leaves_the_rest(cuda, m, n):
    x, w = R.matrix(L, m, 256, "nvfp4", 5, cuda), R.matrix(L, n, 256, "nvfp4", 6, cuda)
    want = L.linear_fp4(x, w)
    pool = torch.full((8 + m * n + 4096,), -7.0, dtype=torch.bfloat16, device=cuda)
    out = pool[8:8 + m * n].view(m, n)
    assert L.linear_fp4(x, w, out=out) is out
    assert torch.equal(out, want)
    assert (pool[:8] == -7).all() and (pool[8 + m * n:] == -7).all()


@pytest.mark.parametrize("m", [0, 4])
def test_empty(cuda, m):
    n = 4 if m == 0 else 0
    for fmt in FORMATS:
        x, w = (L.quantize_fp4(torch.randn((r, 64), device=cuda), fmt) for r in (m, n))
        assert L.linear_fp4(x, w).shape == (m, n)
        assert L.gated_linear_fp4(x, w, w).shape == (m, n)
        d = torch.zeros((m, n), dtype=torch.bfloat16, device=cuda)
        for g, rows in zip(L.linear_fp4_backward(d, x, w), (m, n)):
            assert g.shape == (rows, 64) and not g.any()
        for g, rows in zip(L.gated_linear_fp4_backward(d, d, d, x, w, w), (m, n, n)):
            assert g.shape == (rows, 64) and not g.any()
        assert L.dequantize_fp4(x).shape == (m, 64)


# ------------------------------------------------------------------------------------------------ gated

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 300, 4096), (16, 129, 512), (40, 250, 992), (64, 96, 96), (130, 257, 288),
                                   (300, 640, 1056), (700, 3000, 160)])
def test_gated(cuda, fmt, act, m, n, k):
    x = R.matrix(L, m, k, fmt, m + k, cuda, scale=2.0 ** -2)
    wg, wu = R.matrix(L, n, k, fmt, n + k + 1, cuda, scale=2.0 ** -4), R.matrix(L, n, k, fmt, n + k + 2, cuda, scale=2.0 ** -3)
    xv, gv, uv = R.values(x), R.values(wg), R.values(wu)
    g, u = xv @ gv.t(), xv @ uv.t()
    eg, eu = R.product_bound(xv, gv), R.product_bound(xv, uv)
    want = R.act(g, act) * u
    # act itself: a few fp32 steps of exp, erfc and the division, 2^-18 of act(g) and, through the rounding of
    # exp's argument, of g act'(g) <= 1.2 (1 + |g|) max(act slope terms): covered by 2^-18 (|act| + min(|g|, 8))
    through = (1.13 * eg + 2.0 ** -18 * (R.act(g, act).abs() + g.abs().clamp(max=8.0) * torch.exp(-g.abs() / 2))) * (u.abs() + eu) \
        + R.act(g, act).abs() * eu
    for dtype, half in HALF.items():
        h, hg, hu = L.gated_linear_fp4(x, wg, wu, act, dtype=dtype, save=True)
        close(h, want, (want.abs() + through) * half + through + TINY[dtype])
        close(hg, g, (g.abs() + eg) * half + eg + TINY[dtype])
        close(hu, u, (u.abs() + eu) * half + eu + TINY[dtype])
        assert torch.equal(L.gated_linear_fp4(x, wg, wu, act, dtype=dtype), h)


# --------------------------------------------------------------------------------------------- backward

# The last ones: contractions cut into parts (few tiles, long), and large enough that dg and du are single bf16 values.
GRAD_SHAPES = [(1, 1, 32), (2, 9, 64), (100, 130, 96), (64, 64, 256), (257, 300, 1056), (1000, 513, 288), (300, 2000, 512),
               (4, 6000, 96), (3, 5001, 160), (5000, 40, 64), (2500, 33, 288), (600, 2000, 2048), (601, 2001, 2080)]


def grad_bounds(d, w):
    """|d w| rounding bounds for a contraction of bf16 d with exact w: accumulation in steps of 16."""
    s = d.abs() @ w.abs()
    return (d.shape[1] / 16 + 2) * 2.0 ** -23 * s, s


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
def test_linear_backward(cuda, fmt, m, n, k):
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
    strided = torch.zeros((m, n + 3), dtype=torch.bfloat16, device=cuda)
    strided[:, 2:n + 2] = dy
    for a, b in zip(L.linear_fp4_backward(strided[:, 2:n + 2], x, w), (dx, dw)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
def test_gated_backward(cuda, fmt, act, m, n, k):
    x = R.matrix(L, m, k, fmt, m + k, cuda, scale=2.0 ** -2)
    wg, wu = R.matrix(L, n, k, fmt, n + k + 1, cuda, scale=2.0 ** -4), R.matrix(L, n, k, fmt, n + k + 2, cuda, scale=2.0 ** -3)
    xv, gv, uv = R.values(x), R.values(wg), R.values(wu)
    gen = torch.Generator(device=cuda).manual_seed(m)
    dh, gate, up = ((torch.randn((m, n), generator=gen, device=cuda) * s).to(torch.bfloat16) for s in (1.0, 3.0, 2.0))
    g, u, d = gate.double(), up.double(), dh.double()
    dg, du = d * u * R.act_slope(g, act), d * R.act(g, act)
    # rounding to bf16 (2^-8), and the activation's fp32 steps as in test_gated
    soft = 2.0 ** -18 * (1 + g.abs()).clamp(max=9.0) * d.abs()
    eg, eu = dg.abs() * 2.0 ** -8 + soft * u.abs() * 1.01, du.abs() * 2.0 ** -8 + soft * 1.01
    dx, dwg, dwu = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act)
    for got, pairs in ((dx, ((dg, eg, gv), (du, eu, uv))), (dwg, ((dg.t(), eg.t(), xv),)), (dwu, ((du.t(), eu.t(), xv),))):
        want = sum(a @ b for a, _, b in pairs)
        bound = sum(grad_bounds(a, b)[0] * len(pairs) * 1.01 + e @ b.abs() for a, e, b in pairs)
        close(got, want, (want.abs() + bound) * 2.0 ** -8 + bound)
    only_x, a, b = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(True, False))
    assert a is None and b is None and torch.equal(only_x, dx)
    none, a, b = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act, need=(False, True))
    assert none is None and torch.equal(a, dwg) and torch.equal(b, dwu)


def test_backward_of_unaligned_gradients(cuda):
    """Gradients that start on any element, n a multiple of 8 and not."""
    for m, n in ((40, 136), (40, 133), (700, 264)):
        x, w = R.matrix(L, m, 96, "mxfp4", 1, cuda), R.matrix(L, n, 96, "mxfp4", 2, cuda)
        pool = torch.randn((3, m * n + 8), device=cuda).to(torch.bfloat16)
        for off in (1, 2, 8):
            a, b, c = (t[off:off + m * n].view(m, n) for t in pool)
            copies = [t.clone() for t in (a, b, c)]
            for got, want in zip(L.gated_linear_fp4_backward(a, b, c, x, w, w), L.gated_linear_fp4_backward(*copies, x, w, w)):
                assert torch.equal(got, want)
            for got, want in zip(L.linear_fp4_backward(a, x, w), L.linear_fp4_backward(copies[0], x, w)):
                assert torch.equal(got, want)


@pytest.mark.parametrize("m,n,k", [(1, 200, 96), (7, 6000, 64), (130, 400, 320), (60, 1001, 512)])
def test_gated_backward_of_small_problems_is_as_good_as_one_rounding(cuda, m, n, k):
    """Small problems carry dg and du in two terms: an error of 2^-16 in them, so what is left is the result's rounding."""
    x, wg, wu = (R.matrix(L, r, k, "mxfp4", i, cuda, scale=0.25) for i, r in enumerate((m, n, n)))
    dh, gate, up = (torch.randn((m, n), device=cuda).to(torch.bfloat16) for _ in range(3))
    g, u, d = gate.double(), up.double(), dh.double()
    dg, du = d * u * R.act_slope(g, "silu"), d * R.act(g, "silu")
    want = (dg @ R.values(wg) + du @ R.values(wu), dg.t() @ R.values(x), du.t() @ R.values(x))
    for got, w in zip(L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, "silu"), want):
        assert (got.double() - w).norm() <= 1.05 * (w.to(torch.bfloat16).double() - w).norm()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_gradients_against_differences(cuda, act):
    """<gradient, direction> against the central difference of the 64-bit loss along that direction."""
    m, n, k = 33, 70, 64
    x, wg, wu = (R.matrix(L, r, k, "nvfp4", 10 + i, cuda, scale=s) for i, (r, s) in enumerate(((m, 0.25), (n, 0.1), (n, 0.1))))
    vals = [R.values(t) for t in (x, wg, wu)]
    h, gate, up = L.gated_linear_fp4(x, wg, wu, act, save=True)
    dh = torch.randn((m, n), device=cuda).to(torch.bfloat16)
    grads = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, act)

    def loss(xv, gv, uv):
        return (dh.double() * R.act(xv @ gv.t(), act) * (xv @ uv.t())).sum()

    gen = torch.Generator(device=cuda).manual_seed(1)
    for i in range(3):
        v = torch.randn(vals[i].shape, generator=gen, device=cuda, dtype=torch.float64)
        t = 1e-5
        hi, lo = list(vals), list(vals)
        hi[i], lo[i] = vals[i] + t * v, vals[i] - t * v
        diff = ((loss(*hi) - loss(*lo)) / (2 * t)).item()
        got = (grads[i].double() * v).sum().item()
        # gate, up, dg, du and the result are bf16: five roundings of at most 2^-8, through terms whose absolute
        # sum is this
        a = dh.double().abs()
        g, u = vals[0] @ vals[1].t(), vals[0] @ vals[2].t()
        dg, du = a * u.abs() * 1.13 + a * 0.8 * g.abs() * u.abs(), a * g.abs() * 1.13
        size = {0: dg @ vals[1].abs() + du @ vals[2].abs(), 1: dg.t() @ vals[0].abs(), 2: du.t() @ vals[0].abs()}[i]
        assert abs(got - diff) <= 5 * 2.0 ** -8 * (size * v.abs()).sum().item()
        # independent roundings: far closer than that
        assert abs(got - diff) <= 8 * 2.0 ** -8 * (size * v).norm().item()


# --------------------------------------------------------------------------------- streams, graphs, chain

def _block(x, wg, wu, wd):
    """A feed-forward block as a serving program runs it."""
    h = L.gated_linear_fp4(L.quantize_fp4(x, wg.format), wg, wu, "silu")
    return L.linear_fp4(L.quantize_fp4(h, wd.format), wd)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 17, 150])
def test_feed_forward_block(cuda, fmt, m):
    k, n = 512, 1376
    wg, wu = (R.matrix(L, n, k, fmt, s, cuda, scale=2.0 ** -5) for s in (1, 2))
    wd = R.matrix(L, k, n, fmt, 3, cuda, scale=2.0 ** -5)
    x = torch.randn((m, k), device=cuda).to(torch.bfloat16)
    y = _block(x, wg, wu, wd)
    # each stage against the reference on the values that entered it
    xq = L.quantize_fp4(x, fmt)
    h = L.gated_linear_fp4(xq, wg, wu, "silu")
    xv = R.values(xq)
    want_h = R.act(xv @ R.values(wg).t(), "silu") * (xv @ R.values(wu).t())
    assert (h.double() - want_h).norm() <= 2.0 ** -8 * want_h.norm()
    hv = R.values(L.quantize_fp4(h, fmt))
    want = hv @ R.values(wd).t()
    close(y, want, want.abs() * 2.0 ** -8 + R.product_bound(hv, R.values(wd)) * 1.01)


def test_training_step(cuda):
    """Forward with save, both backward passes chained, gradients of every operand."""
    m, k, n = 96, 256, 352
    fmt = "mxfp4"
    x, wg, wu, wd = (R.matrix(L, r, c, fmt, i, cuda, scale=2.0 ** -3) for i, (r, c) in enumerate(((m, k), (n, k), (n, k), (k, n))))
    h, gate, up = L.gated_linear_fp4(x, wg, wu, "silu", save=True)
    hq = L.quantize_fp4(h, fmt)
    y = L.linear_fp4(hq, wd)
    dy = torch.randn_like(y)
    dh, dwd = L.linear_fp4_backward(dy, hq, wd)
    dx, dwg, dwu = L.gated_linear_fp4_backward(dh, gate, up, x, wg, wu, "silu")
    vals = [R.values(t).requires_grad_(True) for t in (x, wg, wu)]
    hv, wdv = R.values(hq).requires_grad_(True), R.values(wd).requires_grad_(True)
    (hv @ wdv.t() * dy.double()).sum().backward()
    (R.act(vals[0] @ vals[1].t(), "silu") * (vals[0] @ vals[2].t()) * hv.grad).sum().backward()
    for got, want in ((dh, hv.grad), (dwd, wdv.grad), (dx, vals[0].grad), (dwg, vals[1].grad), (dwu, vals[2].grad)):
        # at most six bf16 roundings stand between: each at most 2^-8, 2^-8 / sqrt(3) in the mean square
        assert (got.double() - want).norm() <= 6 * 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("m", [3, 140])
def test_graph_replay_follows_inputs(cuda, m):
    k, n = 256, 520
    wg, wu, wd = (R.matrix(L, r, c, "nvfp4", i, cuda, scale=2.0 ** -4) for i, (r, c) in enumerate(((n, k), (n, k), (k, 544))))
    wd = R.matrix(L, k, n // 32 * 32, "nvfp4", 5, cuda, scale=2.0 ** -4)
    x = torch.randn((m, k), device=cuda).to(torch.bfloat16)

    def step():
        xq = L.quantize_fp4(x, "nvfp4")
        h, g, u = L.gated_linear_fp4(xq, wg, wu, "gelu_tanh", save=True)
        hq = L.quantize_fp4(h[:, :n // 32 * 32], "nvfp4")
        y = L.linear_fp4(hq, wd)
        return (y, *L.linear_fp4_backward(y, hq, wd), *L.gated_linear_fp4_backward(h, g, u, xq, wg, wu, "gelu_tanh"))

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for seed in range(3):
        x.copy_(torch.randn((m, k), generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda))
        want = step()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
    assert L.last_status() == 0


def test_other_streams(cuda):
    x, w = R.matrix(L, 200, 512, "mxfp4", 1, cuda), R.matrix(L, 300, 512, "mxfp4", 2, cuda)
    want = L.linear_fp4(x, w)
    dy = torch.randn((200, 300), device=cuda).to(torch.bfloat16)
    want_g = L.linear_fp4_backward(dy, x, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [(L.linear_fp4(x, w, stream=s), L.linear_fp4_backward(dy, x, w, stream=s)) for s in streams for _ in range(4)]
    got.append((L.linear_fp4(x, w, stream=streams[0].cuda_stream), L.linear_fp4_backward(dy, x, w, stream=streams[1].cuda_stream)))
    torch.cuda.synchronize()
    for y, g in got:
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(g, want_g))


@pytest.mark.parametrize("fmt", FORMATS)
def test_garbage_in_the_row_padding_of_scales(cuda, fmt):
    """Scale rows beyond the matrix may hold anything, NaN included."""
    m, n, k = 70, 200, 352
    nan = 255 if fmt == "mxfp4" else 0x7F
    mats = [R.matrix(L, r, k, fmt, r, cuda, scale=0.25) for r in (m, n)]
    dirty = []
    for q in mats:
        s = q.scales.clone()
        t = s.view(-(-q.rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4)  # [group, row / 32, row % 32, tile, scale]
        rows = torch.arange(t.shape[0] * 128, device=cuda).view(t.shape[0], 4, 32)
        t[rows >= q.rows] = nan
        dirty.append(L.Fp4Matrix(q.codes, s, q.rows, k, fmt, q.tensor_scale))
    dy, g, u = (torch.randn((m, n), device=cuda).to(torch.bfloat16) for _ in range(3))

    def all_of(x, w):
        return (L.dequantize_fp4(x), L.linear_fp4(x, w), L.linear_fp4(w, w), L.gated_linear_fp4(x, w, w), *L.linear_fp4_backward(dy, x, w),
                *L.gated_linear_fp4_backward(dy, g, u, x, w, w))

    for a, b in zip(all_of(*dirty), all_of(*mats)):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_beyond_32_bits(cuda, fmt):
    """More than 2^32 elements in x (quantisation, expansion) and in y and dy (products): the last rows are right."""
    rows, cols = 140000, 32768
    big = torch.zeros((rows, cols), dtype=torch.bfloat16, device=cuda)
    big[-300:] = torch.randn((300, cols), device=cuda).to(torch.bfloat16)
    q = L.quantize_fp4(big, fmt)
    tail = L.quantize_fp4(big[-300:], fmt)
    assert torch.equal(q.codes[-300:], tail.codes) and not q.codes[:-300].any()
    L.dequantize_fp4(q, out=big)
    assert torch.equal(big[-300:], L.dequantize_fp4(tail, dtype=torch.bfloat16))
    del q
    k = 64
    x, w = R.matrix(L, rows, k, fmt, 1, cuda), R.matrix(L, cols, k, fmt, 2, cuda)
    xv = R.values(L.Fp4Matrix.from_rows(x.codes[-300:], x.scale_rows()[-300:], fmt, x.tensor_scale))
    wv = R.values(w)
    L.linear_fp4(x, w, out=big)
    want = xv @ wv.t()
    close(big[-300:], want, want.abs() * 2.0 ** -8 + R.product_bound(xv, wv) * 1.01)
    L.gated_linear_fp4(x, w, w, out=big)
    want = R.act(want, "silu") * want
    assert (big[-300:].double() - want).norm() <= 2.0 ** -8 * want.norm()
    big.zero_()
    big[-300:] = torch.randn((300, cols), device=cuda).to(torch.bfloat16)
    dx, dw = L.linear_fp4_backward(big, x, w)
    d = big[-300:].double()
    for got, a, b in ((dx[-300:], d, wv), (dw, d.t(), xv)):
        want, s = a @ b, a.abs() @ b.abs()
        # the rows before are zeros: the sums take as many steps, of which only the last add anything
        close(got, want, want.abs() * 2.0 ** -8 + (a.shape[1] / 16 + 2) * 2.0 ** -23 * s * 1.01)
    assert not dx[:-300].any()


def test_infinite_gradients_stay_in_their_rows_and_columns(cuda):
    m, n, k = 40, 96, 64
    x, w = R.matrix(L, m, k, "mxfp4", 1, cuda), R.matrix(L, n, k, "mxfp4", 2, cuda)
    dy = torch.randn((m, n), device=cuda).to(torch.bfloat16)
    clean = L.linear_fp4_backward(dy, x, w)
    dy[3, 5] = float("inf")
    dx, dw = L.linear_fp4_backward(dy, x, w)
    rows = torch.arange(m, device=cuda) != 3
    cols = torch.arange(n, device=cuda) != 5
    assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dw[cols], clean[1][cols])
    assert not torch.isfinite(dx[3]).any() and not torch.isfinite(dw[5]).any()


def test_repeated_calls_give_the_same_bits(cuda):
    x, w = R.matrix(L, 9, 4096, "nvfp4", 1, cuda), R.matrix(L, 1000, 4096, "nvfp4", 2, cuda)
    dy = torch.randn((9, 1000), device=cuda).to(torch.bfloat16)
    first = (L.linear_fp4(x, w), L.gated_linear_fp4(x, w, w), *L.linear_fp4_backward(dy, x, w))
    for _ in range(10):
        for a, b in zip((L.linear_fp4(x, w), L.gated_linear_fp4(x, w, w), *L.linear_fp4_backward(dy, x, w)), first):
            assert torch.equal(a, b)
