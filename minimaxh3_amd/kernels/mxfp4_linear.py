"""Linear layers on microscaled 4-bit floating point (an extension; no counterpart in the reference's files).

Beside the FP8 linears: weights and activations in blocks of 32 e2m1 values (+-{0, 1/2, 1, 3/2, 2, 3, 4,
6}) under a shared power of two (the OCP MX FP4 format), half the bytes of FP8 and a product that runs
on the matrix cores' 4-bit rate, twice the 8-bit one.  Activations are quantized on the fly.

Codes are [rows, K / 2] uint8, two a byte with the even column low; scales are [ceil(K / 256), rows, 8]
uint8, the exponent + 127 of each block (255: the block held an infinity or NaN and reads as NaN).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops
from .fp8_linear import ACT_GELU_TANH, ACT_NONE, _convert_blocks, apply_lora_adapters


def quantize_mxfp4(x2d: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] bf16 / fp16 / fp32, K % 32 == 0 -> (codes, scales).  A block's power of two puts its
    largest magnitude into [3.5, 7); values round to the nearest code, ties to the even one, and those
    above 6 become 6."""
    if x2d.ndim != 2 or not x2d.is_cuda:
        raise ValueError("quantize_mxfp4 expects a 2D CUDA tensor")
    return ops.mxfp4_quant(x2d)


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [M, K] that ``quantize_mxfp4``'s codes and scales stand for (exact in bf16 and fp32)."""
    return ops.mxfp4_dequant(codes, scales, dtype)


class MXFP4Linear(nn.Module):
    """nn.Linear replacement with 4-bit weights (buffers ``w4``, ``w_scale``, ``bias``; K % 32 == 0).

    The output is bf16(act(x w^T + bias)) with one rounding, in the input's dtype.  ``adapters`` holds
    LoRA triples as ``FP8Linear`` does; they and the activation then run after the product as torch
    ops, in the input's dtype (``forward_quantized``: bf16).  Code that attaches adapters to
    ``nn.Linear`` and ``FP8Linear`` by type has to be told of this class.

    The fp32 sum's order depends on the size of the product: a token's output may differ in its last
    bit between a call of a few tokens and one of many (``mxf8_gemm_mxfp4`` in include/mxf8.h)."""

    def __init__(self, in_features: int, out_features: int) -> None:
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.adapters: list[tuple[torch.Tensor, torch.Tensor, float]] = []
        self.act = ACT_NONE

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "MXFP4Linear":
        """Quantize ``linear``'s weight and free it."""
        weight = linear.weight.detach()
        if not weight.is_cuda:
            weight = weight.cuda()
        mod = cls.from_quantized(*quantize_mxfp4(weight), linear.bias)
        if isinstance(getattr(linear, "adapters", None), list):
            mod.adapters = list(linear.adapters)
        linear.weight = None
        linear.bias = None
        return mod

    @classmethod
    @torch.no_grad()
    def from_quantized(cls, w4: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                       device: torch.device | str | None = None) -> "MXFP4Linear":
        """MXFP4Linear from stored buffers: codes ``w4 [N, K / 2]``, ``w_scale`` and an optional bias [N]
        (stored as bf16), as ``from_linear`` computes them."""
        if w4.dtype != torch.uint8 or w4.ndim != 2 or w4.shape[1] == 0 or w4.shape[1] % 16:
            raise ValueError("from_quantized: w4 must be uint8 [N, K / 2] with K a multiple of 32")
        N, K = w4.shape[0], 2 * w4.shape[1]
        if w_scale.dtype != torch.uint8 or tuple(w_scale.shape) != ops.mxfp4_scale_shape(N, K):
            raise ValueError(f"from_quantized: w_scale must be uint8 {ops.mxfp4_scale_shape(N, K)}")
        if bias is not None and bias.numel() != N:
            raise ValueError(f"from_quantized: bias must hold {N} values")
        dev = torch.device(device) if device is not None else w4.device
        mod = cls(K, N)
        mod.register_buffer("w4", w4.to(dev).contiguous())
        mod.register_buffer("w_scale", w_scale.to(dev).contiguous())
        mod.register_buffer("bias", None if bias is None else bias.detach().to(dev, torch.bfloat16).reshape(N).contiguous())
        return mod

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x2d = x if x.ndim == 2 else x.reshape(-1, self.in_features)
        out = ops.mxfp4_linear(x2d, self.w4, self.w_scale, self.bias, ACT_NONE if self.adapters else int(self.act))
        if x.dtype != torch.bfloat16:
            out = out.to(x.dtype)
        if self.adapters:
            out = self._adapted(x2d, out)
        return out if x.ndim == 2 else out.reshape(*x.shape[:-1], self.out_features)

    def forward_quantized(self, x4: torch.Tensor, x_scale: torch.Tensor,
                          x_modulated: torch.Tensor | None = None) -> torch.Tensor:
        """``forward`` on an input quantized already (``quantize_mxfp4``, ``gated_residual_norm``) ->
        bf16 [M, N].  LoRA adapters read the unquantized input ``x_modulated`` [..., K]."""
        if x4.ndim != 2 or 2 * x4.shape[1] != self.in_features:
            raise ValueError(f"forward_quantized: expected 4-bit codes [M, {self.in_features // 2}]")
        if not self.adapters:
            return ops.gemm_mxfp4(x4, self.w4, x_scale, self.w_scale, self.bias, int(self.act))
        if x_modulated is None:
            raise ValueError("forward_quantized: LoRA adapters need the unquantized input (x_modulated)")
        out = ops.gemm_mxfp4(x4, self.w4, x_scale, self.w_scale, self.bias, ACT_NONE)
        return self._adapted(x_modulated.reshape(-1, self.in_features), out)

    def _adapted(self, x2d: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        out = apply_lora_adapters(x2d, out, self.adapters)
        return torch.nn.functional.gelu(out, approximate="tanh") if self.act == ACT_GELU_TANH else out

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, act={self.act}"


def convert_transformer_to_mxfp4(transformer: nn.Module, exclude_patterns: str | list[str], keep_edge_blocks: int,
                                 fuse_gelu: bool = False) -> int:
    """``convert_transformer_to_fp8`` with ``MXFP4Linear``: the same blocks and exclusions, for linears whose
    in_features are a multiple of 32 and out_features of 16.  Returns the number of converted modules."""
    return _convert_blocks(transformer, exclude_patterns, keep_edge_blocks, fuse_gelu, MXFP4Linear, 32)
