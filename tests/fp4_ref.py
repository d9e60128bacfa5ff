"""64-bit reference of the microscaled 4-bit formats and of the operators on them (test infrastructure).

Written from the definitions; runs on whatever device its tensors are on."""
import math

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAG = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def e4m3_values(device="cpu"):
    """The 127 finite non-negative e4m3 values, by byte."""
    b = torch.arange(127, dtype=torch.float64, device=device)
    e, m = torch.div(b, 8, rounding_mode="floor"), torch.remainder(b, 8)
    return torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e - 7))


def nearest_even(v, grid):
    """Index of the nearest grid value to v >= 0 (ties to the even index, above the last: the last)."""
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(v, mid, right=False), torch.bucketize(v, mid, right=True)
    return torch.where((lo != hi) & (lo % 2 == 1), hi, lo)


def quantize(x, fmt, ts=None):
    """x [rows, k] float -> (codes [rows, k/2], scale bytes [rows, k/block])."""
    rows, k = x.shape
    block = BLOCK[fmt]
    t = x.float()
    if fmt == "nvfp4" and ts is not None:
        inv = 1.0 / ts.float() if float(ts) != 0.0 else torch.zeros_like(ts)
        t = t * inv
    finite = torch.isfinite(t).view(rows, k // block, block).all(-1)
    t = torch.where(torch.isfinite(t), t, torch.zeros_like(t)).double().view(rows, k // block, block)
    amax = t.abs().amax(-1)
    if fmt == "mxfp4":
        # floor(log2) by exponent: frexp gives amax = f 2^e with f in [1/2, 1)
        e = torch.frexp(amax)[1].double() - 1
        byte = torch.where(amax > 0, (e - 2 + 127).clamp(min=0), torch.zeros_like(e))
        scale = torch.exp2(byte - 127)
        byte = torch.where(finite, byte, torch.full_like(byte, 255))
    else:
        grid = e4m3_values(x.device)
        byte = nearest_even(amax, grid * 6)  # nearest to amax / 6, without the division
        scale = grid[byte]
        byte = torch.where(finite, byte, torch.full_like(byte, 0x7F))
    mag = torch.tensor(MAG, dtype=torch.float64, device=x.device)
    idx = nearest_even(t.abs() / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(-1), mag)
    idx = torch.where((scale > 0).unsqueeze(-1), idx, torch.zeros_like(idx))
    code = (idx + 8 * torch.signbit(t)).to(torch.uint8).view(rows, k)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.to(torch.uint8), finite


def scale_values(byte, fmt):
    if fmt == "mxfp4":
        return torch.where(byte == 255, torch.nan, torch.exp2(byte.double() - 127))
    grid = torch.cat((e4m3_values(byte.device), torch.full((1,), torch.nan, dtype=torch.float64, device=byte.device)))
    return grid[byte.long()]


def values(q):
    """The numbers an Fp4Matrix stands for, float64."""
    rows, k = q.shape
    codes = torch.stack((q.codes & 15, q.codes >> 4), dim=-1).view(rows, k).long()
    mag = torch.tensor(MAG + tuple(-v for v in MAG), dtype=torch.float64, device=codes.device)
    v = mag[codes] * scale_values(q.scale_rows(), q.format).repeat_interleave(BLOCK[q.format], dim=1)
    return v if q.tensor_scale is None else v * q.tensor_scale.double()


def act(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return g * torch.special.ndtr(g)
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def act_slope(g, kind):
    g = g.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act(g, kind).sum(), g)[0]


def matrix(L, rows, k, fmt, seed, device, scale=1.0, ts=True):
    """A random Fp4Matrix: codes of all sixteen kinds, scales spread over several binades."""
    gen = torch.Generator(device="cpu").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, k // 2), generator=gen, dtype=torch.uint8)
    blocks = k // BLOCK[fmt]
    if fmt == "mxfp4":
        sb = (127 + math.log2(scale) + torch.randint(-3, 2, (rows, blocks), generator=gen)).round().to(torch.uint8)
        tensor_scale = None
    else:
        sb = torch.randint(0x28, 0x48, (rows, blocks), generator=gen, dtype=torch.uint8)  # 2^-2 .. 3.75
        tensor_scale = torch.tensor([scale * 0.7], dtype=torch.float32, device=device) if ts else None
    return L.Fp4Matrix.from_rows(codes.to(device), sb.to(device), fmt, tensor_scale)


def product_bound(x, w, step_products=16):
    """Bound on the fp32 accumulation error of x w^T: one rounding (2^-23 of the running magnitude, truncation
    included) for each `step_products` products and one for the scaling, never above sum |x||w| each."""
    k = x.shape[1]
    return (k / step_products + 2) * 2.0 ** -23 * (x.abs() @ w.abs().t())
