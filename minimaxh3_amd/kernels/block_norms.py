"""What stands between two branches of a DiT block (an extension; no counterpart in the reference's files).

The attention's or the MLP's output is gated into the residual stream, perhaps after a norm of its own,
and the sum is normed and modulated for the next branch's linear.  ``gated_residual_norm`` does it in one
pass over the rows and can hand the result to ``FP8Linear.forward_quantized`` or
``MXFP4Linear.forward_quantized`` in their own formats.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .. import ops

_QUANT = {None: N.QUANT_NONE, "e4m3": N.QUANT_E4M3, "mxfp4": N.QUANT_MXFP4}


def gated_residual_norm(
    x: torch.Tensor,
    branch: torch.Tensor | None,
    gate: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    *,
    branch_weight: torch.Tensor | None = None,
    weight: torch.Tensor | None = None,
    norm: str = "layer",
    eps: float = 1e-6,
    residual_scale: float = 1.0,
    quantize: str | None = None,
    return_modulated: bool = False,
):
    """(r, y) of a residual stream x and a branch's output, both [B, S, C]:

        u = branch, or with ``branch_weight`` [C] its RMS norm times that
        r = residual_scale * x + gate * u
        y = norm(r) * weight * (1 + scale) + shift       (norm: "layer" or "rms", over C)

    gate, shift and scale hold a row per batch item, [B, C], or one per S / G consecutive tokens (a
    frame), [B, G, C]; each may be None (1, 0, 0), and so may ``weight`` [C].  All tensors have x's
    dtype: bf16, fp16 or fp32.  Arithmetic is fp32, y is taken from the unrounded r, and each output is
    rounded once; a token's results do not depend on the others of the call, to the bit.  With
    ``branch=None`` r is x itself (residual_scale must be 1): the norm before a model's first branch.
    C <= 16384.

    ``quantize="e4m3"`` returns (r, x8 [B S, C], x_scale [B S, 1]) for ``FP8Linear.forward_quantized``,
    ``quantize="mxfp4"`` (r, x4 [B S, C / 2], x_scale [ceil(C / 256), B S, 8]) for
    ``MXFP4Linear.forward_quantized``: the codes that ``quantize_rows`` / ``quantize_mxfp4`` give for y,
    bit for bit, without y's way through memory; ``return_modulated`` appends y [B, S, C] (LoRA
    adapters need it).
    """
    if norm not in ("layer", "rms"):
        raise ValueError(f'gated_residual_norm: norm must be "layer" or "rms", got {norm!r}')
    if quantize not in _QUANT:
        raise ValueError(f'gated_residual_norm: quantize must be None, "e4m3" or "mxfp4", got {quantize!r}')
    if branch is None and residual_scale != 1.0:
        raise ValueError("gated_residual_norm: residual_scale needs a branch")
    r, y, codes, scales = ops.gated_residual_norm(
        x, branch, gate, shift, scale, branch_weight, weight, norm == "layer", float(eps), float(residual_scale),
        _QUANT[quantize], bool(return_modulated))
    if branch is None:
        r = x
    if quantize is None:
        return r, y
    return (r, codes, scales, y) if return_modulated else (r, codes, scales)
