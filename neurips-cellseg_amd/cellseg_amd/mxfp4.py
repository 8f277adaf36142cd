"""``mxfp4_quantize`` / ``mxfp4_linear`` - microscaled 4-bit numbers (OCP MX, MXFP4) and the linear layer on them, next to the fp8 mode.

32 consecutive values of the last axis share one power-of-two scale (e8m0); each value is e2m1: 0, 0.5, 1, 1.5, 2, 3, 4 or 6 and a sign,
4.25 bits a value in all.  ``mxfp4_linear`` rounds its input the same way and multiplies both on the 4-bit matrix instructions with float32
sums (csrc/kernels_mxfp4.hip).  For serving: an input that wants a gradient, or carries a forward-mode tangent, is refused.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib
from .head_losses import TYPES, _pitch, rows_of

BLOCK = 32


class MXFP4Tensor:
    """``codes`` uint8 [..., 16 * blocks] (two e2m1 codes a byte, the even one in the low half), ``scales`` uint8 [..., blocks] (2^(s - 127);
    255: NaN), blocks = ceil(width / 32); the last block of a row is filled up with zeros.  ``dtype``: what ``dequantize`` gives."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, width: int, dtype: torch.dtype = torch.bfloat16):
        blocks = -(-int(width) // BLOCK)
        if width < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() < 1 or codes.shape[-1] != 16 * blocks \
                or tuple(scales.shape) != tuple(codes.shape[:-1]) + (blocks,):
            raise ValueError(f"expected uint8 codes [..., {16 * blocks}] and scales [..., {blocks}] for a width of {width}, got {codes.dtype} {tuple(codes.shape)} "
                             f"and {scales.dtype} {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        if dtype not in TYPES:
            raise TypeError(f"dtype is bfloat16, float16 or float32, got {dtype}")
        self.codes, self.scales, self.width, self.dtype = codes.contiguous(), scales.contiguous(), int(width), dtype
        if self.codes.data_ptr() % 16:
            self.codes = self.codes.clone()

    @property
    def shape(self) -> Tuple[int, ...]:
        return tuple(self.codes.shape[:-1]) + (self.width,)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values, rounded once to ``dtype`` (default: the type that was quantised)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in TYPES:
            raise TypeError(f"dtype is bfloat16, float16 or float32, got {dtype}")
        _lib.require_gpu(self.codes)
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _lib.on_device(self.device):
            check(lib.cs_mxfp4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), out.numel() // self.width, self.width, TYPES[dtype],
                                          out.data_ptr(), _lib.raw_stream(self.device)), "cs_mxfp4_dequantize")
        return out

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={self.shape}, dtype={self.dtype}, device={self.device})"


def _no_grad(x: torch.Tensor, name: str) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient: detach its input or call it under torch.no_grad()")
    if forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"{name} has no forward-mode derivative: detach its input")


def mxfp4_quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x [..., width] (bfloat16, float16 or float32) -> its MXFP4 form.  A block that holds an infinity or a NaN becomes NaN."""
    _no_grad(x, "mxfp4_quantize")
    if x.dtype not in TYPES:
        raise TypeError(f"mxfp4_quantize takes bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected x [..., width], got {tuple(x.shape)}")
    _lib.require_gpu(x)
    rows, width = rows_of(x), x.shape[-1]
    blocks = -(-width // BLOCK)
    codes = torch.empty(tuple(x.shape[:-1]) + (16 * blocks,), dtype=torch.uint8, device=x.device)
    scales = torch.empty(tuple(x.shape[:-1]) + (blocks,), dtype=torch.uint8, device=x.device)
    with _lib.on_device(x.device):
        check(lib.cs_mxfp4_quantize(rows.data_ptr(), _pitch(rows), rows.shape[0], width, TYPES[x.dtype], codes.data_ptr(),
                                    scales.data_ptr(), _lib.raw_stream(x.device)), "cs_mxfp4_quantize")
    return MXFP4Tensor(codes, scales, width, x.dtype)


def mxfp4_linear(x: torch.Tensor, weight: MXFP4Tensor) -> torch.Tensor:
    """``mxfp4(x) @ weight.T``: x [..., width], weight [outputs, width] -> [..., outputs] in x's type, float32 sums, one rounding."""
    _no_grad(x, "mxfp4_linear")
    if not isinstance(weight, MXFP4Tensor):
        raise TypeError(f"weight is an MXFP4Tensor (mxfp4_quantize makes one), got {type(weight).__name__}")
    if x.dtype not in TYPES:
        raise TypeError(f"mxfp4_linear takes bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or len(weight.shape) != 2 or x.shape[-1] != weight.width:
        raise ValueError(f"expected x [..., {weight.width}] and weight [outputs, {weight.width}], got {tuple(x.shape)} and {weight.shape}")
    if not x.is_cuda:
        _lib.require_gpu(x)
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    rows, outputs = rows_of(x), weight.shape[0]
    y = torch.empty(tuple(x.shape[:-1]) + (outputs,), dtype=x.dtype, device=x.device)
    with _lib.on_device(x.device):
        size = lib.cs_mxfp4_linear_workspace_bytes(rows.shape[0], weight.width, outputs)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        check(lib.cs_mxfp4_linear(rows.data_ptr(), _pitch(rows), rows.shape[0], weight.width, TYPES[x.dtype], weight.codes.data_ptr(), weight.scales.data_ptr(), outputs,
                                  y.data_ptr(), ws.data_ptr() if size else None, size, _lib.raw_stream(x.device)), "cs_mxfp4_linear")
    return y
