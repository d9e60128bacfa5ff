"""PyTorch operator binding over the C ABI.

    import int4linear_b200.torch_op            # registers the ops
    y = torch.ops.int4linear.linear(x_packed, w_packed)     # [m, k/2] u8, [n, k/2] u8 -> [m, n] i32
    z = torch.ops.int4linear.linear_scaled(x_packed, w_packed, row_scale, col_scale, bias)   # -> [m, n] bf16
    p = torch.ops.int4linear.pack(values)                   # [m, n] i8/i32 -> [m, ceil(n/8)] i32
    c, s = torch.ops.int4linear.quantize_fp4(x, "mxfp4", None)              # [m, k] floats -> codes [m, k/2] u8, scales u8
    y = torch.ops.int4linear.linear_fp4(xc, xs, None, wc, ws, None, bias, "mxfp4")                # -> [m, n] bf16
    h = torch.ops.int4linear.gated_linear_fp4(xc, xs, None, gc, gs, None, uc, us, None, "silu", "mxfp4")   # -> [m, n] bf16

The ops run on the tensors' device and the current CUDA stream, have shape-inference ("fake")
implementations so they trace under FakeTensor / torch.compile graphs, and have no CPU kernels:
the operator exists only as the sm_100a library.  This is the natural caller of the launcher the
reference exposes as linear_v21_launch (kernels/linear_v21.h:760) on a PyTorch stack; the
reference itself has no Python binding.
"""
from __future__ import annotations

import torch

from . import fp4 as _fp4
from .linear import linear as _linear_fn
from .linear import linear_scaled as _linear_scaled_fn
from .packer import pack_device as _pack_device


@torch.library.custom_op("int4linear::linear", mutates_args=(), device_types="cuda")
def linear(x_packed: torch.Tensor, w_packed: torch.Tensor) -> torch.Tensor:
    return _linear_fn(x_packed, w_packed)


@linear.register_fake
def _(x_packed, w_packed):
    if x_packed.dim() != 2 or w_packed.dim() != 2:
        raise ValueError("int4linear::linear expects 2-D packed operands")
    bx = x_packed.shape[1] * x_packed.element_size()
    bw = w_packed.shape[1] * w_packed.element_size()
    if bx != bw:
        raise ValueError("packed operands disagree on K")
    return x_packed.new_empty((x_packed.shape[0], w_packed.shape[0]), dtype=torch.int32)


@torch.library.custom_op("int4linear::linear_scaled", mutates_args=(), device_types="cuda")
def linear_scaled(x_packed: torch.Tensor, w_packed: torch.Tensor, row_scale: torch.Tensor | None,
                  col_scale: torch.Tensor | None, bias: torch.Tensor | None) -> torch.Tensor:
    """bf16((X @ W^T) * row_scale[:, None] * col_scale[None, :] + bias): the dequantising epilogue of
    int4_linear_scaled_launch_async.  Scales and bias are float32 CUDA vectors or None."""
    return _linear_scaled_fn(x_packed, w_packed, row_scale, col_scale, bias)


@linear_scaled.register_fake
def _(x_packed, w_packed, row_scale, col_scale, bias):
    if x_packed.dim() != 2 or w_packed.dim() != 2:
        raise ValueError("int4linear::linear_scaled expects 2-D packed operands")
    if x_packed.shape[1] * x_packed.element_size() != w_packed.shape[1] * w_packed.element_size():
        raise ValueError("packed operands disagree on K")
    return x_packed.new_empty((x_packed.shape[0], w_packed.shape[0]), dtype=torch.bfloat16)


@torch.library.custom_op("int4linear::pack", mutates_args=(), device_types="cuda")
def pack(values: torch.Tensor) -> torch.Tensor:
    return _pack_device(values)


@pack.register_fake
def _(values):
    return values.new_empty((values.shape[0], (values.shape[1] + 7) // 8), dtype=torch.int32)


def _matrix(codes, scales, tensor_scale, format):
    return _fp4.Fp4Matrix(codes, scales, codes.shape[0], codes.shape[1] * 2, format, tensor_scale)


@torch.library.custom_op("int4linear::quantize_fp4", mutates_args=(), device_types="cuda")
def quantize_fp4(x: torch.Tensor, format: str, tensor_scale: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of fp4.quantize_fp4."""
    q = _fp4.quantize_fp4(x, format, tensor_scale)
    return q.codes, q.scales


@quantize_fp4.register_fake
def _(x, format, tensor_scale):
    if x.dim() != 2:
        raise ValueError("int4linear::quantize_fp4 expects a 2-D tensor")
    rows, k = x.shape
    _fp4._check_shape(rows, k, format)
    return x.new_empty((rows, k // 2), dtype=torch.uint8), x.new_empty((_fp4._scale_bytes(rows, k, format),), dtype=torch.uint8)


@torch.library.custom_op("int4linear::linear_fp4", mutates_args=(), device_types="cuda")
def linear_fp4(x_codes: torch.Tensor, x_scales: torch.Tensor, x_tensor_scale: torch.Tensor | None,
               w_codes: torch.Tensor, w_scales: torch.Tensor, w_tensor_scale: torch.Tensor | None,
               bias: torch.Tensor | None, format: str) -> torch.Tensor:
    """bf16 X @ W^T + bias of two microscaled matrices (fp4.linear_fp4)."""
    return _fp4.linear_fp4(_matrix(x_codes, x_scales, x_tensor_scale, format), _matrix(w_codes, w_scales, w_tensor_scale, format), bias)


@linear_fp4.register_fake
def _(x_codes, x_scales, x_tensor_scale, w_codes, w_scales, w_tensor_scale, bias, format):
    if x_codes.dim() != 2 or w_codes.dim() != 2 or x_codes.shape[1] != w_codes.shape[1]:
        raise ValueError("int4linear::linear_fp4 expects 2-D codes that agree in k")
    return x_codes.new_empty((x_codes.shape[0], w_codes.shape[0]), dtype=torch.bfloat16)


@torch.library.custom_op("int4linear::gated_linear_fp4", mutates_args=(), device_types="cuda")
def gated_linear_fp4(x_codes: torch.Tensor, x_scales: torch.Tensor, x_tensor_scale: torch.Tensor | None,
                     gate_codes: torch.Tensor, gate_scales: torch.Tensor, gate_tensor_scale: torch.Tensor | None,
                     up_codes: torch.Tensor, up_scales: torch.Tensor, up_tensor_scale: torch.Tensor | None,
                     activation: str, format: str) -> torch.Tensor:
    """bf16 act(X @ Wg^T) * (X @ Wu^T) (fp4.gated_linear_fp4)."""
    return _fp4.gated_linear_fp4(_matrix(x_codes, x_scales, x_tensor_scale, format),
                                 _matrix(gate_codes, gate_scales, gate_tensor_scale, format),
                                 _matrix(up_codes, up_scales, up_tensor_scale, format), activation)


@gated_linear_fp4.register_fake
def _(x_codes, x_scales, x_tensor_scale, gate_codes, gate_scales, gate_tensor_scale, up_codes, up_scales, up_tensor_scale,
      activation, format):
    if not (x_codes.dim() == gate_codes.dim() == up_codes.dim() == 2) or gate_codes.shape != up_codes.shape or \
            x_codes.shape[1] != gate_codes.shape[1]:
        raise ValueError("int4linear::gated_linear_fp4 expects 2-D codes that agree in k, and weights of one shape")
    return x_codes.new_empty((x_codes.shape[0], gate_codes.shape[0]), dtype=torch.bfloat16)
