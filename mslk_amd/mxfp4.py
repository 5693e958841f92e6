"""Linear layers in microscaled 4-bit floating point (MXFP4): quantizer, products, gated feed-forward, experts.

The operators are `torch.ops.mslk.quantize_mxfp4`, `dequantize_mxfp4`, `mxfp4_mm`, `mxfp4_gated_mm` and `mxfp4_grouped_mm` (GPU
kernels only, native: csrc/torch_ops.cpp; csrc/mx_quantize.hip, mx_gemm.hip); the functions below are their Python form.  They have
no counterpart in the reference's FP8 path: they are its layers with half the bytes of weights and twice the matrix rate.

A row of K values (K a multiple of 32) is K / 32 blocks: 32 e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and a power
of two.  Codes are bytes [.., K / 2] with the earlier value in the low half (uint8, or torch.float4_e2m1fn_x2, which is the same), scales
bytes s [.., K / 32] that stand for 2^(s - 127), 255 for NaN (uint8 or torch.float8_e8m0fnu): the layouts of the OCP microscaling
specification, so weights quantized elsewhere can be used as they are.  Products take both operands so, sum in fp32 and round once.

Nothing here is differentiable.  Codes have to be contiguous.  Both tensors of scales are copied in each call, into another order, where they cannot be
read as they lie (K no multiple of 512, of 128 for products of few tiles, or scales that do not begin on 16 bytes; up to 32 rows and as many columns as
32 per compute unit are read from anywhere) and where the product is large enough to gain by it (2 M N K of 1.1e12 operations and more).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

_library = torch.library.Library("mslk", "FRAGMENT")


def _fake_quantize(a):
    return tuple(torch.empty((*a.shape[:-1], a.shape[-1] // n), dtype=torch.uint8, device=a.device) for n in (2, 32))


def _fake_dequantize(codes, scales, out_dtype=None):
    return torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=out_dtype or torch.bfloat16, device=codes.device)


def _fake_mm(XQ, WQ, x_scale, w_scale, bias=None, out_dtype=None):
    return torch.empty((*XQ.shape[:-1], WQ.shape[0]), dtype=out_dtype or torch.bfloat16, device=XQ.device)


def _fake_gated(XQ, WQ, x_scale, w_scale, out_dtype=None):
    return torch.empty((*XQ.shape[:-1], WQ.shape[0] // 2), dtype=out_dtype or torch.bfloat16, device=XQ.device)


def _fake_grouped(XQ, WQ, x_scale, w_scale, M_sizes, gated=False, out_dtype=None):
    return torch.empty((XQ.shape[0], WQ.shape[1] // (2 if gated else 1)), dtype=out_dtype or torch.bfloat16, device=XQ.device)


_OPS = {
    "quantize_mxfp4": ("(Tensor a) -> (Tensor, Tensor)", _fake_quantize),
    "dequantize_mxfp4": ("(Tensor codes, Tensor scales, ScalarType? out_dtype=None) -> Tensor", _fake_dequantize),
    "mxfp4_mm": ("(Tensor XQ, Tensor WQ, Tensor x_scale, Tensor w_scale, Tensor? bias=None, ScalarType? out_dtype=None) -> Tensor", _fake_mm),
    "mxfp4_gated_mm": ("(Tensor XQ, Tensor WQ, Tensor x_scale, Tensor w_scale, ScalarType? out_dtype=None) -> Tensor", _fake_gated),
    "mxfp4_grouped_mm": ("(Tensor XQ, Tensor WQ, Tensor x_scale, Tensor w_scale, Tensor M_sizes, bool gated=False, "
                         "ScalarType? out_dtype=None) -> Tensor", _fake_grouped),
}
for _name, (_schema, _fake) in _OPS.items():
    if not hasattr(torch.ops.mslk, _name):
        _library.define(_name + _schema)
        torch.library.register_fake(f"mslk::{_name}", _fake, lib=_library)
    # Outside of autograd: without a derivative its fallback would make the results part of the graph of any input that requires a
    # gradient.
    _library.impl(_name, torch.library.fallthrough_kernel, "Autograd")


def _check_gpu(name: str, *tensors: torch.Tensor) -> None:
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError(f"mslk_amd.{name}: inputs must be GPU tensors (no CPU implementation)")


def quantize_mxfp4(a: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows a [.., K] (bf16, fp16, fp32) -> codes [.., K / 2] and scales [.., K / 32], both uint8.

    Of a block's largest magnitude m the scale is 2^(floor(log2 m) - 2), at least 2^-127; values are rounded to nearest even, those
    beyond 6 scales to 6.  A block with a NaN or an infinity becomes NaN: scale 255, codes 0."""
    _check_gpu("quantize_mxfp4", a)
    return torch.ops.mslk.quantize_mxfp4(a)


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What codes and scales stand for: exact in bf16 and fp32 up to the largest finite number, rounded in fp16."""
    _check_gpu("dequantize_mxfp4", codes)
    return torch.ops.mslk.dequantize_mxfp4(codes, scales, out_dtype)


def mxfp4_mm(XQ: torch.Tensor, WQ: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Y [.., N] = X W^T + bias of codes XQ [.., K / 2], WQ [N, K / 2] and their scales; `bias` [N] in fp32 or bf16, Y in bf16 or fp16."""
    _check_gpu("mxfp4_mm", XQ, WQ)
    return torch.ops.mslk.mxfp4_mm(XQ, WQ, x_scale, w_scale, bias, out_dtype)


def mxfp4_gated_mm(XQ: torch.Tensor, WQ: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
                   out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Y [.., N] = silu(X Wg^T) * (X Wu^T): both projections of a gated feed-forward block, with its activation.  WQ [2 N, K / 2] holds
    the N rows of the gate, then the N rows of the other projection."""
    _check_gpu("mxfp4_gated_mm", XQ, WQ)
    return torch.ops.mslk.mxfp4_gated_mm(XQ, WQ, x_scale, w_scale, out_dtype)


def mxfp4_grouped_mm(XQ: torch.Tensor, WQ: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor, M_sizes: torch.Tensor,
                     gated: bool = False, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The products of a router's experts: the first M_sizes[0] rows of XQ [total_M, K / 2] times WQ[0]^T, the next M_sizes[1] times
    WQ[1]^T, ...; `gated`: each as in `mxfp4_gated_mm`.  M_sizes [G] (int64) is read on the GPU only, so a captured graph follows it;
    rows beyond the sum of the sizes are left uninitialised."""
    _check_gpu("mxfp4_grouped_mm", XQ, WQ)
    return torch.ops.mslk.mxfp4_grouped_mm(XQ, WQ, x_scale, w_scale, M_sizes, gated, out_dtype)
