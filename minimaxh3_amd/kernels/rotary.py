"""Rotary positions over several axes (an extension; no counterpart in the reference's files).

A video DiT turns the query and key heads between its QKV projection and its attention, each pair of
channels by an angle that grows with the token's time, row or column, usually after an RMS norm of the
head.  ``rotary_table`` makes the cos / sin of a sequence's angles, once per resolution and length;
``rotate_qk`` norms and turns q and k, reading the projection's views and writing each value once, in a
layout that ``fp8_attention`` takes.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

from .. import ops


def rotary_table(positions: torch.Tensor, axis_dims: Sequence[int], theta: float = 10000.0) -> torch.Tensor:
    """cos / sin pairs [..., P, 2] fp32 of positions [..., A] on a GPU.

    Axis a takes ``axis_dims[a]`` (even) channels of a head, ``axis_dims[a] / 2`` pairs; the pairs of
    all axes follow each other, P = sum(axis_dims) / 2 <= 256 of them.  Pair i of axis a has the angle
    ``positions[..., a] * theta ** (-2 i / axis_dims[a])``.  Positions are int32, int64, fp32 or fp64
    (fractions of a frame are fine); the angle is formed and reduced in 64 bits, so far positions lose
    nothing.  1 to 4 axes.
    """
    return ops.rotary_table(positions, [int(d) for d in axis_dims], float(theta))


def rotate_qk(q: torch.Tensor, k: torch.Tensor | None, table: torch.Tensor, q_weight: torch.Tensor | None = None,
              k_weight: torch.Tensor | None = None, eps: float = 1e-6,
              interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS-normed (per head, where a weight is given) and rotated q [B, H, S, D] and k [B, Hk, S, D].

    table [S, P, 2], or [B, S, P, 2] for positions that differ between items, from ``rotary_table``.
    The pairs are channels (2 j, 2 j + 1), or (j, j + P) with ``interleaved=False``; channels from 2 P
    on pass through.  q_weight / k_weight [D] in q's dtype: ``x / sqrt(mean(x^2) + eps) * weight``
    over the head's D channels first.  bf16, fp16 or fp32, in any strides; fp32 arithmetic, rounded
    once.  Hk may differ from H, and k may be None.  The results are new tensors with the dimensions in
    the inputs' memory order, so the [B, S, H, D] views of a projection stay such views.
    """
    qo, ko = ops.rotate_qk(q, k, table, q_weight, k_weight, float(eps), bool(interleaved))
    return qo, None if k is None else ko
