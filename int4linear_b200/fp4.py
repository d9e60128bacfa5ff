"""Microscaled 4-bit floating point: quantisation, the linear layer and the gated feed-forward block on it,
and their backward passes.

    xq = quantize_fp4(x)                                   # [m, k] floats -> Fp4Matrix
    y  = linear_fp4(xq, wq, bias)                          # x w^T + bias, bf16 or fp16
    h  = gated_linear_fp4(xq, wq_gate, wq_up, "silu")      # act(x wg^T) * (x wu^T), one kernel
    h, gate, up = gated_linear_fp4(..., save=True)         # training: the products are kept
    dx, dw = linear_fp4_backward(dy, xq, wq)
    dx, dwg, dwu = gated_linear_fp4_backward(dh, gate, up, xq, wq_gate, wq_up, "silu")

Two formats: "mxfp4" (blocks of 32, power-of-two scales) and "nvfp4" (blocks of 16, e4m3 scales, one float per
matrix besides).  Like the integer operators these exist only as sm_100a kernels: there is no CPU implementation.
All calls are asynchronous on `stream` (default: the current one of the operands' device) and can be captured into
CUDA graphs after a first call on the device; memory they allocate belongs to that stream.  The reference has
integer operands only, so none of these has a counterpart there.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

from . import _lib
from .linear import Int4LinearError

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCKS = {"mxfp4": 32, "nvfp4": 16}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


class _CMatrix(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("tensor_scale", ctypes.c_void_p),
                ("rows", ctypes.c_int), ("k", ctypes.c_int), ("format", ctypes.c_int)]


def _scale_bytes(rows: int, k: int, fmt: str) -> int:
    block = BLOCKS[fmt]
    return -(-rows // 128) * -(-k // (4 * block)) * 512


def _check_shape(rows: int, k: int, fmt: str) -> None:
    if fmt not in FORMATS:
        raise ValueError(f"unknown format {fmt!r}: expected one of {sorted(FORMATS)}")
    if rows < 0 or k <= 0 or k % 32 != 0:
        raise ValueError("need k > 0 and k % 32 == 0")
    if rows > 2 ** 26 or k > 2 ** 26:
        raise ValueError("rows and k are at most 2^26")


def _check_tensor_scale(ts, fmt: str, device) -> None:
    import torch
    if ts is None:
        return
    if fmt != "nvfp4":
        raise ValueError("tensor_scale belongs to nvfp4")
    if not isinstance(ts, torch.Tensor) or ts.dtype != torch.float32 or ts.numel() != 1 or ts.device != device:
        raise ValueError("tensor_scale must be a float32 tensor of one element on the matrix's device")


@dataclass(frozen=True, eq=False)
class Fp4Matrix:
    """A quantised [rows, k] matrix.

    codes: uint8 [rows, k/2], low nibble = even index.  scales: uint8, 1-D, in the tensor core's order: tiles of
    128 rows x 4 scales (512 bytes, scale (r, j) at byte (r % 32) * 16 + (r // 32) * 4 + j), along k first, rows
    padded to 128 and scales to 4 (the padding along k must not be NaN; 0 is right).  `from_rows` builds it from
    scales in row order, `scale_rows` gives them back.  tensor_scale: nvfp4 only, float32 CUDA tensor of one
    element or None (1).  The tensors are held, not copied: the matrix changes with their values (their memory must stay
    theirs: no resize_ or set_)."""
    codes: "torch.Tensor"  # noqa: F821
    scales: "torch.Tensor"  # noqa: F821
    rows: int
    k: int
    format: str = "mxfp4"
    tensor_scale: "torch.Tensor | None" = None  # noqa: F821
    device: "torch.device" = field(init=False, repr=False)  # noqa: F821
    _c: _CMatrix = field(init=False, repr=False)
    _p: int = field(init=False, repr=False)  # address of _c

    def __post_init__(self):
        import torch
        _check_shape(self.rows, self.k, self.format)
        c, s = self.codes, self.scales
        if not c.is_cuda or c.dtype != torch.uint8 or tuple(c.shape) != (self.rows, self.k // 2) or not c.is_contiguous():
            raise ValueError("codes must be a contiguous CUDA uint8 tensor [rows, k/2]")
        if s.device != c.device or s.dtype != torch.uint8 or s.dim() != 1 or not s.is_contiguous() or \
                s.numel() != _scale_bytes(self.rows, self.k, self.format):
            raise ValueError("scales must be a contiguous 1-D uint8 tensor of "
                             f"{_scale_bytes(self.rows, self.k, self.format)} bytes on the codes' device")
        _check_tensor_scale(self.tensor_scale, self.format, c.device)
        if c.data_ptr() % 16 or s.data_ptr() % 16:
            raise ValueError("codes and scales must start on 16-byte boundaries")
        self._wrap()

    def _wrap(self):
        ts = self.tensor_scale
        d = self.__dict__  # (frozen for users; this is part of the construction)
        d["device"] = self.codes.device
        d["_c"] = c = _CMatrix(self.codes.data_ptr(), self.scales.data_ptr(), ts.data_ptr() if ts is not None else None,
                               self.rows, self.k, FORMATS[self.format])
        d["_p"] = ctypes.addressof(c)

    @classmethod
    def _new(cls, rows: int, k: int, fmt: str, tensor_scale, device) -> "Fp4Matrix":
        """An uninitialised matrix, its arguments already checked."""
        import torch
        q = object.__new__(cls)
        q.__dict__.update(codes=torch.empty(rows, k // 2, dtype=torch.uint8, device=device),
                          scales=torch.empty(_scale_bytes(rows, k, fmt), dtype=torch.uint8, device=device),
                          rows=rows, k=k, format=fmt, tensor_scale=tensor_scale)
        q._wrap()
        return q

    def __reduce__(self):  # copies and pickles are built anew: _c holds addresses
        return type(self), (self.codes, self.scales, self.rows, self.k, self.format, self.tensor_scale)

    @property
    def shape(self):
        return (self.rows, self.k)

    @classmethod
    def from_rows(cls, codes, scale_rows, format: str = "mxfp4", tensor_scale=None) -> "Fp4Matrix":
        """From codes [rows, k/2] and scale bytes in row order, [rows, k/block] (uint8, or a 1-byte float type)."""
        import torch
        rows, k = codes.shape[0], codes.shape[1] * 2
        _check_shape(rows, k, format)
        if scale_rows.element_size() != 1 or tuple(scale_rows.shape) != (rows, k // BLOCKS[format]):
            raise ValueError("scale_rows must hold one byte per block: [rows, k/block]")
        sb = scale_rows.contiguous().view(torch.uint8)
        rt, kt = -(-rows // 128), -(-sb.shape[1] // 4)
        full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=sb.device)
        full[:rows, :sb.shape[1]] = sb
        tiled = full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
        return cls(codes.contiguous(), tiled, rows, k, format, tensor_scale)

    def scale_rows(self):
        """The scale bytes in row order, [rows, k/block] uint8."""
        blocks = self.k // BLOCKS[self.format]
        rt, kt = -(-self.rows // 128), -(-blocks // 4)
        full = self.scales.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)
        return full[:self.rows, :blocks].contiguous()


def _where(device, stream, inputs):
    """(stream handle, context to work in or None) of one call.  The context makes the device and stream current, so
    that allocations belong to them; none is needed where they already are."""
    import torch
    if stream is None:
        index = device.index
        handle = torch._C._cuda_getCurrentRawStream(index)
        return handle, None if torch.cuda.current_device() == index else torch.cuda.device(device)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device != device:
        raise ValueError("stream belongs to another device than the operands")
    current = torch.cuda.current_stream(device)
    if stream != current:
        for t in inputs():  # their memory must not be handed out again before this stream is done with it
            if t is not None:
                t.record_stream(stream)
    elif torch.cuda.current_device() == device.index:
        return stream.cuda_stream, None
    return stream.cuda_stream, torch.cuda.stream(stream)


def _run(body, device, stream, inputs):
    """body(handle) on the call's device and stream."""
    handle, ctx = _where(device, stream, inputs)
    if ctx is None:
        return body(handle)
    with ctx:
        return body(handle)


_types: dict = {}  # torch type -> INT4L_TYPE_*, filled by the first call


def _type_of(dtype) -> int:
    if not _types:
        import torch
        _types.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2})
    t = _types.get(dtype)
    if t is None:
        raise TypeError(f"expected bfloat16, float16 or float32, not {dtype}")
    return t


def _parts(*mats):
    return [t for q in mats for t in (q.codes, q.scales, q.tensor_scale)]


def _check(st: int, where: str) -> None:
    if st != 0:
        raise Int4LinearError(st, where)


def _check_out(out, shape, dtype, device, name="out"):
    if tuple(out.shape) != shape or out.dtype != dtype or not out.is_contiguous() or out.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on the operands' device")


def _wanted_format(format: str | None, out: Fp4Matrix | None) -> str:
    if out is None:
        return "mxfp4" if format is None else format
    if format is not None and format != out.format:
        raise ValueError(f"out is {out.format}, not {format}")
    return out.format


def quantize_fp4(x, format: str | None = None, tensor_scale=None, out: Fp4Matrix | None = None, stream=None) -> Fp4Matrix:
    """Quantise a CUDA matrix [rows, k] of bfloat16, float16 or float32 (k % 32 == 0; rows may be strided).
    `format`: "mxfp4" or "nvfp4"; None is that of `out`, or "mxfp4".

    mxfp4: scale 2^(floor(log2 amax) - 2) per 32 elements.  nvfp4: the values are multiplied by 1 / tensor_scale,
    scale = amax / 6 rounded to e4m3 per 16 elements.  Codes are rounded to nearest, ties to even, and saturate
    at 6.  A block that holds a NaN or an infinity becomes NaN.  `out`: a matrix of that shape and format to write
    into; its own tensor_scale is then used."""
    if not x.is_cuda or x.dim() != 2:
        raise ValueError("quantize_fp4 expects a 2-D CUDA tensor; there is no CPU implementation")
    rows, k = x.shape
    device = x.device
    t = _type_of(x.dtype)
    format = _wanted_format(format, out)
    if out is not None:
        if out.shape != (rows, k) or out.device != device or tensor_scale is not None:
            raise ValueError("out must have the shape and device of x, and brings its own tensor_scale")
    else:
        _check_shape(rows, k, format)
        if tensor_scale is not None:
            _check_tensor_scale(tensor_scale, format, device)

    def body(handle):
        src = x
        pitch = x.stride(0) if rows > 1 else k
        if x.stride(1) != 1 or pitch < k:
            src, pitch = x.contiguous(), k
        q = out if out is not None else Fp4Matrix._new(rows, k, format, tensor_scale, device)
        if rows:
            _check(_lib.load().int4_linear_fp4_quantize_async(src.data_ptr(), t, pitch, q._p, handle), "int4_linear_fp4_quantize_async")
        return q

    return _run(body, device, stream, lambda: (x, tensor_scale) if out is None else (x, *_parts(out)))


def dequantize_fp4(q: Fp4Matrix, dtype=None, out=None, stream=None):
    """The values of a quantised matrix, [rows, k] float32 (or `dtype`: bfloat16, float16)."""
    import torch
    if dtype is None:
        dtype = out.dtype if out is not None else torch.float32
    t = _type_of(dtype)
    if out is not None:
        _check_out(out, q.shape, dtype, q.device)

    def body(handle):
        y = out if out is not None else torch.empty(q.rows, q.k, dtype=dtype, device=q.device)
        if q.rows:
            _check(_lib.load().int4_linear_fp4_dequantize_async(q._p, y.data_ptr(), t, handle), "int4_linear_fp4_dequantize_async")
        return y

    return _run(body, q.device, stream, lambda: (*_parts(q), out))


def _check_operands(x: Fp4Matrix, *ws: Fp4Matrix) -> tuple[int, int]:
    rows = ws[0].rows
    for w in ws:
        if w.k != x.k or w.format != x.format or w.device != x.device or w.rows != rows:
            raise ValueError("operands must agree in k, format and device (and both weights in their rows)")
    return x.rows, rows


def _half(dtype, out):
    """(output type, its INT4L_TYPE_ number)"""
    import torch
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16
    if dtype is torch.bfloat16:
        return dtype, 0
    if dtype is torch.float16:
        return dtype, 1
    raise ValueError("the output is bfloat16 or float16")


def _check_act(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: expected one of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[activation]


def linear_fp4(x: Fp4Matrix, w: Fp4Matrix, bias=None, out=None, dtype=None, stream=None):
    """Y = X @ W^T (+ bias): [m, n] bfloat16 (default) or float16, accumulated in fp32 and rounded once.
    `bias`: float32 CUDA vector of n elements."""
    import torch
    m, n = _check_operands(x, w)
    dtype, t = _half(dtype, out)
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (n,) or bias.device != x.device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous float32 tensor with {n} elements on the operands' device")
    if out is not None:
        _check_out(out, (m, n), dtype, x.device)

    def body(handle):
        y = out if out is not None else torch.empty(m, n, dtype=dtype, device=x.device)
        if m and n:
            _check(_lib.load().int4_linear_fp4_launch_async(x._p, w._p, bias.data_ptr() if bias is not None else None, y.data_ptr(),
                                                            t, handle), "int4_linear_fp4_launch_async")
        return y

    return _run(body, x.device, stream, lambda: (*_parts(x, w), bias, out))


def gated_linear_fp4(x: Fp4Matrix, w_gate: Fp4Matrix, w_up: Fp4Matrix, activation: str = "silu", out=None, dtype=None,
                     save: bool = False, stream=None):
    """H = act(X @ Wg^T) * (X @ Wu^T), both products, the activation and the multiplication in one kernel.

    activation: "silu", "gelu" or "gelu_tanh".  Returns H, [m, n] bfloat16 (default) or float16; with `save`
    (H, gate, up), the products rounded to the same type; gated_linear_fp4_backward takes them in bfloat16."""
    import torch
    m, n = _check_operands(x, w_gate, w_up)
    dtype, t = _half(dtype, out)
    act = _check_act(activation)
    if out is not None:
        _check_out(out, (m, n), dtype, x.device)

    def body(handle):
        h = out if out is not None else torch.empty(m, n, dtype=dtype, device=x.device)
        gate, up = (torch.empty_like(h), torch.empty_like(h)) if save else (None, None)
        if m and n:
            _check(_lib.load().int4_linear_fp4_gated_launch_async(
                x._p, w_gate._p, w_up._p, act, h.data_ptr(), gate.data_ptr() if save else None, up.data_ptr() if save else None,
                t, handle), "int4_linear_fp4_gated_launch_async")
        return (h, gate, up) if save else h

    return _run(body, x.device, stream, lambda: (*_parts(x, w_gate, w_up), out))


def _terms_flag(terms: int | None) -> int:
    if terms not in (None, 1, 2):
        raise ValueError("terms is 1, 2 or None")
    return {None: 0, 1: 1 << 8, 2: 1 << 9}[terms]


def _check_grad(t, m: int, n: int, device, name: str):
    import torch
    if t.dtype != torch.bfloat16 or tuple(t.shape) != (m, n) or t.device != device:
        raise ValueError(f"{name} must be a bfloat16 tensor of shape [{m}, {n}] on the operands' device")


def _workspace(m, n, k, gated, want_x, want_w, device):
    import torch
    need = _lib.load().int4_linear_fp4_grad_workspace_bytes(m, n, k, gated, int(want_x), int(want_w))
    return torch.empty(max(need, 256), dtype=torch.uint8, device=device)


def linear_fp4_backward(grad_y, x: Fp4Matrix, w: Fp4Matrix, need=(True, True), stream=None):
    """(dX, dW) = (dY @ W, dY^T @ X) in bfloat16, with respect to the values the operands stand for (a bias's gradient is
    grad_y.sum(0)).  grad_y: bfloat16 [m, n].  `need` leaves one out (None in its place)."""
    import torch
    m, n = _check_operands(x, w)
    _check_grad(grad_y, m, n, x.device, "grad_y")
    want_x, want_w = bool(need[0]), bool(need[1])

    def body(handle):
        empty = m == 0 or n == 0  # an empty sum is 0
        new = torch.zeros if empty else torch.empty
        dx = new(m, x.k, dtype=torch.bfloat16, device=x.device) if want_x else None
        dw = new(n, x.k, dtype=torch.bfloat16, device=x.device) if want_w else None
        if not empty and (want_x or want_w):
            dy = grad_y.contiguous()
            if dy.data_ptr() % 16:
                dy = dy.clone()
            ws = _workspace(m, n, x.k, 0, want_x, want_w, x.device)
            _check(_lib.load().int4_linear_fp4_grad_async(
                dy.data_ptr(), x._p, w._p, dx.data_ptr() if want_x else None, dw.data_ptr() if want_w else None,
                ws.data_ptr(), ws.numel(), handle), "int4_linear_fp4_grad_async")
        return dx, dw

    return _run(body, x.device, stream, lambda: (grad_y, *_parts(x, w)))


def gated_linear_fp4_backward(grad_h, gate, up, x: Fp4Matrix, w_gate: Fp4Matrix, w_up: Fp4Matrix, activation: str = "silu",
                              need=(True, True), stream=None, terms: int | None = None):
    """(dX, dWg, dWu) of gated_linear_fp4 in bfloat16, with respect to the values the operands stand for.

    gate, up: the products kept by a forward pass in bfloat16, [m, n] like grad_h.
    dG = dH up act'(gate), dU = dH act(gate); dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X.
    `need` = (input, weights) leaves gradients out (None in their place).
    `terms`: 1 rounds dG and dU to bfloat16 (results then have 1.4 times the error of one rounding), 2 carries them as two
    bfloat16 terms (one rounding) in products of twice the length (4096 x 14336 x 4096: 1.6 and 3.3 ms).  None lets the sizes decide: two terms where that
    takes a few microseconds at most or m n <= 65536.  Give it where the bits of a token's gradient must not depend on the number
    of tokens beside it in that way."""
    import torch
    m, n = _check_operands(x, w_gate, w_up)
    act = _check_act(activation)
    for t, name in ((grad_h, "grad_h"), (gate, "gate"), (up, "up")):
        _check_grad(t, m, n, x.device, name)
    want_x, want_w = bool(need[0]), bool(need[1])
    flag = _terms_flag(terms)

    def body(handle):
        empty = m == 0 or n == 0
        new = torch.zeros if empty else torch.empty
        dx = new(m, x.k, dtype=torch.bfloat16, device=x.device) if want_x else None
        dwg = new(n, x.k, dtype=torch.bfloat16, device=x.device) if want_w else None
        dwu = new(n, x.k, dtype=torch.bfloat16, device=x.device) if want_w else None
        if not empty and (want_x or want_w):
            dh, g, u = grad_h.contiguous(), gate.contiguous(), up.contiguous()
            ws = _workspace(m, n, x.k, 1 | flag, want_x, want_w, x.device)
            _check(_lib.load().int4_linear_fp4_gated_grad_async(
                dh.data_ptr(), g.data_ptr(), u.data_ptr(), x._p, w_gate._p, w_up._p, act | flag, dx.data_ptr() if want_x else None,
                dwg.data_ptr() if want_w else None, dwu.data_ptr() if want_w else None, ws.data_ptr(), ws.numel(), handle),
                "int4_linear_fp4_gated_grad_async")
        return dx, dwg, dwu

    return _run(body, x.device, stream, lambda: (grad_h, gate, up, *_parts(x, w_gate, w_up)))
