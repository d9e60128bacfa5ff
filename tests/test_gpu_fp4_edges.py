"""GPU: microscaled 4-bit operators where a value is hard to get right.

Activations are read through operands that pass them on unchanged (identity matrices), so every bound is one on a value."""
import math

import pytest
import torch

import fp4_ref as R
import int4linear_b200 as L

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def eye(rows, k, fmt, device):
    """The rows x k identity."""
    codes = torch.zeros((rows, k), dtype=torch.uint8)
    codes[torch.arange(min(rows, k)), torch.arange(min(rows, k))] = 2  # 1
    one = 127 if fmt == "mxfp4" else 0x38
    sb = torch.full((rows, k // R.BLOCK[fmt]), one, dtype=torch.uint8)
    return L.Fp4Matrix.from_rows((codes[:, 0::2] | (codes[:, 1::2] << 4)).to(device), sb.to(device), fmt)


def constant(rows, k, code, fmt, device):
    one = 127 if fmt == "mxfp4" else 0x38
    return L.Fp4Matrix.from_rows(torch.full((rows, k // 2), 17 * code, dtype=torch.uint8, device=device),
                                 torch.full((rows, k // R.BLOCK[fmt]), one, dtype=torch.uint8, device=device), fmt)


def exponent(g, act):
    """The argument whose exponential carries act(g)'s smallness."""
    if act == "silu":
        return g.abs()
    if act == "gelu":
        return g * g / 2
    return 2 * math.sqrt(2 / math.pi) * (g.abs() + 0.044715 * g.abs() ** 3)


def relative(g, act):
    """Relative error of the fp32 arithmetic: the exponential's 2 + 1.173 |a| units in the last place, its argument's roundings
    (at most five of half a unit, so 2.5 |a|), the fitted tail's 1.2e-6 (10 units of 2^-23), a division and the products around
    them (at most 4)."""
    return (16 + 4 * exponent(g, act)) * 2.0 ** -23


def value(g, act):
    """act(g) in 64 bits (gelu by erfc: 1 + erf, and torch's ndtr with it, has lost the lower tail at -8)."""
    return g * torch.special.erfc(-g / math.sqrt(2)) / 2 if act == "gelu" else R.act(g, act)


def slope(g, act):
    """act'(g) in 64 bits, and the sum of the magnitudes of its terms."""
    if act == "silu":
        s, c = torch.sigmoid(g), torch.sigmoid(-g)
        return s * (1 + g * c), s * (1 + (g * c).abs())
    if act == "gelu":
        p, d = torch.special.erfc(-g / math.sqrt(2)) / 2, g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        return p + d, p + d.abs()
    near = g.clamp(-1e3, 1e3)  # (farther out the slope is 0 or 1)
    z = 2 * math.sqrt(2 / math.pi) * (near + 0.044715 * near ** 3)
    s, c = torch.sigmoid(z), torch.sigmoid(-z)
    t = near * c * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * near ** 2)
    return s * (1 + t), s * (1 + t.abs())


@pytest.mark.parametrize("m", [32, 96])
@pytest.mark.parametrize("act,top", [("silu", 1.0), ("silu", 16.0), ("gelu", 1.0), ("gelu", 2.0), ("gelu_tanh", 1.0)])
def test_activation_is_within_one_rounding_everywhere(cuda, m, act, top):
    """g = each value of w_gate (x is the identity, up is 1), down to where act(g) leaves the output type."""
    n, k = 1000, 96
    gen = torch.Generator().manual_seed(m)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    sb = torch.randint(0x18, 0x41, (n, k // 16), generator=gen, dtype=torch.uint8)  # 2^-4 .. 2.25
    wg = L.Fp4Matrix.from_rows(codes.to(cuda), sb.to(cuda), "nvfp4", torch.tensor([top], device=cuda))
    x, up = eye(m, k, "nvfp4", cuda), constant(n, k, 2, "nvfp4", cuda)
    g = R.values(wg)[:, :m].t()  # (exact: at most 6 bits times a power of two)
    assert 6.0 * top <= g.abs().max() <= 13.5 * top
    want = value(g, act)
    for dtype, half in HALF.items():
        h, gate, u = L.gated_linear_fp4(x, wg, up, act, dtype=dtype, save=True)
        assert torch.equal(gate.double(), g) and (u == 1).all()
        err = (h.double() - want).abs()
        # (results and intermediates below 2^-126 have fewer bits)
        bound = want.abs() * (half + relative(g, act) * (1 + half)) + TINY[dtype] + (1 + g.abs()) * 2.0 ** -146
        if act != "gelu":  # 1 / (1 + exp(-v)) is 0 where the divisor passes 2^126: the factor of g is below 2^-126 there
            bound += torch.where(exponent(g, act) > 126 * math.log(2), g.abs() * 2.0 ** -126, torch.zeros_like(g))
        worst = ((err - bound) / want.abs().clamp(min=2.0 ** -140)).max().item()
        assert (err <= bound).all(), worst


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gate_gradients_far_out(cuda, act):
    """dg and du come through identity weights: dx = dg with w_gate = 1, w_up = 0, and dx = du the other way round."""
    n = 128
    g = torch.cat((torch.linspace(-13, 13, 3 * n - 24), torch.tensor([0.0, -0.0, -40.0, 40.0, -86.0, -90.0, 90.0, -1e3, 1e3, 1e5, -1e5, 1e9, -1e9]),
                   torch.tensor([-1.2e13, -5e13, 5e13, 1e15, -1e15, 3e19, -3e19, 1e25, -1e25, 1e38, -1e38]))).view(3, n)
    g = g.to(torch.bfloat16).to(cuda)
    one = torch.ones_like(g)
    x, w, zero = eye(3, n, "mxfp4", cuda), eye(n, n, "mxfp4", cuda), constant(n, n, 0, "mxfp4", cuda)
    dg, _, _ = L.gated_linear_fp4_backward(one, g, one, x, w, zero, act, need=(True, False))
    du, _, _ = L.gated_linear_fp4_backward(one, g, one, x, zero, w, act, need=(True, False))
    gd = g.double()
    small = (1 + gd.abs().clamp(max=100)) * 2.0 ** -133  # (the second term of dg and du is a bf16 too)
    far = gd.clamp(-200, 200)  # (the exponential is 0 in fp32 beyond)
    tail = (far.abs() + 1) * 2.0 ** -140
    want, size = slope(gd, act)
    rel = relative(far, act).clamp(max=2.0 ** -12)
    # A second term carries the rounding of dg and du down to 2^-16.
    err = (dg.double() - want).abs()
    assert torch.isfinite(dg).all() and (err <= want.abs() * 2.0 ** -8 + size * (rel + 2.0 ** -16) * 1.01 + small + tail).all(), err.max()
    want = torch.where(gd < -1e3, torch.zeros_like(gd), torch.where(gd > 1e3, gd, value(gd.clamp(-1e3, 1e3), act)))
    err = (du.double() - want).abs()
    assert torch.isfinite(du).all() and (err <= want.abs() * (2.0 ** -8 + (rel + 2.0 ** -16) * 1.01) + small + tail).all(), err.max()


def test_nan_gate_stays_nan(cuda):
    for act in ("silu", "gelu", "gelu_tanh"):
        n = 64
        g = torch.zeros((2, n), dtype=torch.bfloat16, device=cuda)
        g[1, 5] = float("nan")
        one = torch.ones_like(g)
        x, w = eye(2, n, "mxfp4", cuda), eye(n, n, "mxfp4", cuda)
        dx, dwg, dwu = L.gated_linear_fp4_backward(one, g, one, x, w, w, act)
        assert torch.isnan(dx[1]).all() and torch.isfinite(dx[0]).all()
        for d in (dwg, dwu):
            assert torch.isnan(d[5]).all() and torch.isfinite(d[:5]).all() and torch.isfinite(d[6:]).all()


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 11)])
def test_dequantize_rounds_once(cuda, dtype, bits):
    """Tensor scales for which code x scale x tensor scale lies beside a tie of the 16-bit type, nearer to it than half a step of
    fp32: a product that is rounded to fp32 first lands on the tie and then goes to the even side, right or wrong."""
    mant = {c * (1 + s / 8) for c in (1.0, 1.5) for s in range(8)}
    gen = torch.Generator().manual_seed(bits)
    picks = []
    for _ in range(400):
        p = (1 + torch.randint(0, 2 ** (bits - 1), (1,), generator=gen).item() * 2.0 ** (1 - bits) + 2.0 ** -bits)  # a tie in [1, 2)
        a = sorted(mant)[torch.randint(0, len(mant), (1,), generator=gen).item()]
        ts = torch.tensor([p / a], dtype=torch.float64).float()
        exact = ts.double().item() * a  # 6 bits times 24: exact in 64
        rounded = torch.tensor(exact, dtype=torch.float64).float().double().item()
        if rounded == p and exact != p:
            lo, hi = p - 2.0 ** -bits, p + 2.0 ** -bits
            picks.append((a, ts, lo if exact < p else hi))
    assert len(picks) >= 20
    wrong = 0
    for a, ts, want in picks:
        mags = [(c, s) for c in range(1, 8) for s in range(0x38, 0x40) if R.MAG[c] * R.e4m3_values()[s].item() == a]
        c, s = mags[0]
        q = L.Fp4Matrix.from_rows(torch.full((1, 16), c | (c << 4) | 0x80, dtype=torch.uint8, device=cuda),
                                  torch.full((1, 2), s, dtype=torch.uint8, device=cuda), "nvfp4", ts.to(cuda))
        got = L.dequantize_fp4(q, dtype=dtype).double().view(-1)
        wrong += int((got[0::2] != want).any()) + int((got[1::2] != -want).any())
    assert wrong == 0, f"{wrong} of {2 * len(picks)} values rounded twice"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ts", [0.0, math.inf, -math.inf, math.nan, 3.0e38, -0.37, 1e-38, 2.0 ** -140])
def test_dequantize_under_extreme_tensor_scales(cuda, dtype, ts):
    q = R.matrix(L, 40, 96, "nvfp4", 4, cuda)
    sb = q.scale_rows()
    sb[3, 2] = 0x7F
    q = L.Fp4Matrix.from_rows(q.codes, sb, "nvfp4", torch.tensor([ts], device=cuda))
    want = R.values(q)
    got = L.dequantize_fp4(q, dtype=dtype).double()
    # What rounds beyond the largest value is infinite; products of 64-bit values never overflow before.
    top = (2 - 2.0 ** (-7 if dtype == torch.bfloat16 else -10)) * 2.0 ** (127 if dtype == torch.bfloat16 else 15)
    half_step = top * HALF[dtype] / 2
    want = torch.where(want.abs() >= top + half_step, torch.copysign(torch.full_like(want, math.inf), want), want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.equal(torch.signbit(got[torch.isinf(want)]), torch.signbit(want[torch.isinf(want)]))
    assert ((got - want).abs()[fine] <= want.abs()[fine] * HALF[dtype] + TINY[dtype]).all()


# The second takes the form in which the operands are expanded by a launch of their own.
@pytest.mark.parametrize("m,n,k", [(70, 200, 96), (1030, 4100, 1056)])
def test_nan_block_under_a_tensor_scale_of_zero(cuda, m, n, k):
    """NaN times 0 is NaN in the products and in the expansion, so it is in the gradients."""
    def with_nan(rows, seed, row, block):
        q = R.matrix(L, rows, k, "nvfp4", seed, cuda)
        sb = q.scale_rows()
        sb[row, block] = 0x7F
        return L.Fp4Matrix.from_rows(q.codes, sb, "nvfp4", torch.zeros(1, device=cuda))

    x, w = with_nan(m, 1, m - 1, 2), with_nan(n, 2, n - 1, 4)
    dy = torch.randn((m, n), device=cuda).to(torch.bfloat16)
    dx, dw = L.linear_fp4_backward(dy, x, w)
    y = L.linear_fp4(x, w)
    assert torch.isnan(y[m - 1]).all() and torch.isnan(y[:, n - 1]).all() and not y[:m - 1, :n - 1].any()
    for d, at in ((dx, 4), (dw, 2)):
        hit = torch.zeros(k, dtype=torch.bool, device=cuda)
        hit[16 * at:16 * at + 16] = True
        assert torch.isnan(d[:, hit]).all() and not d[:, ~hit].any()
    gdx, dwg, dwu = L.gated_linear_fp4_backward(dy, dy, dy, x, w, w)
    for d, at in ((gdx, 4), (dwg, 2), (dwu, 2)):
        hit = torch.zeros(k, dtype=torch.bool, device=cuda)
        hit[16 * at:16 * at + 16] = True
        assert torch.isnan(d[:, hit]).all() and not d[:, ~hit].any()
