"""The operators around the FP8 kernels of a DiT block, in 64 bits (test infrastructure only): rotary
positions over several axes, the gated residual with its norms, and 4-bit blocks.

Written from the definitions.  Functions that a kernel's 32-bit arithmetic follows within rounding return
the bound of that rounding beside the result, from the terms of the sums (see each docstring); the rounding
to the output's type comes on top (`half_step`).
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative

# step between neighbours (relative) and smallest subnormal of the output types
_TYPES = {"bf16": (2.0 ** -7, 2.0 ** -133), "fp16": (2.0 ** -10, 2.0 ** -24), "fp32": (2.0 ** -23, 2.0 ** -149)}


def half_step(ref, dtype: str):
    """The most that rounding to nearest moves a value."""
    eps, tiny = _TYPES[dtype]
    return np.abs(ref) * eps / 2 + tiny / 2


def rotary_table(pos, axis_dims, theta: float):
    """pos [..., A] -> [..., P, 2]."""
    pos = np.asarray(pos, np.float64)
    angle = np.concatenate([pos[..., a: a + 1] * theta ** (-2.0 * np.arange(d // 2) / d)
                            for a, d in enumerate(axis_dims)], -1)
    return np.stack([np.cos(angle), np.sin(angle)], -1)


def rotate(x, table, weight=None, eps: float = 1e-6, interleaved: bool = True):
    """x [B, H, S, D], table [S, P, 2] or [B, S, P, 2] -> (result, bound of fp32 arithmetic).

    The norm: a sum of squares in 8 steps and 6 levels, a division, a square root, a reciprocal and two
    products, under 14 / 2 + 5 roundings of the value; the rotation: two products and a sum.  16 U of
    |a| + |b| covers both."""
    x = np.asarray(x, np.float64)
    y = x
    if weight is not None:
        y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    table = np.asarray(table, np.float64)
    t = table if table.ndim == 3 else table[:, None]
    P = table.shape[-2]
    first = np.arange(P) * 2 if interleaved else np.arange(P)
    second = first + (1 if interleaved else P)
    a, b, c, s = y[..., first], y[..., second], t[..., 0], t[..., 1]
    out, bound = y.copy(), 16 * U * np.abs(y)
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    bound[..., first] = bound[..., second] = 16 * U * (np.abs(a) + np.abs(b))
    return out, bound


def _rows(mod, B, S):
    """Modulation rows [B, C] or [B, G, C] spread over the tokens, [B, S, C]."""
    mod = np.asarray(mod, np.float64)
    if mod.ndim == 2:
        mod = mod[:, None]
    return np.repeat(mod, S // mod.shape[1], 1)


def gated_residual_norm(x, branch, gate=None, shift=None, scale=None, branch_weight=None, weight=None,
                        norm: str = "layer", eps: float = 1e-6, residual_scale: float = 1.0):
    """(r, y, bound of r, bound of y), [B, S, C] each.

    A row's sums run over at most 48 elements of one thread, 6 levels between the lanes of a wave and the
    parts of up to 8 waves, under 62 roundings and those of the products' sum: a relative error of under
    g = 80 U in a sum of squares, and of g mean|r| in the mean.  u then has g / 2 + 6 U, r adds a
    product and a sum.  y: the errors of r and of the mean times rstd, g / 2 + 6 U of n, and a rounding for
    each further product and sum."""
    g = 80 * U
    x = np.asarray(x, np.float64)
    B, S, C = x.shape
    r, br = residual_scale * x, 2 * U * np.abs(residual_scale * x)
    if branch is not None:
        u = np.asarray(branch, np.float64)
        du = 0.0
        if branch_weight is not None:
            u = u / np.sqrt(np.mean(u * u, -1, keepdims=True) + eps) * np.asarray(branch_weight, np.float64)
            du = g / 2 + 6 * U
        if gate is not None:
            u = u * _rows(gate, B, S)
        r = r + u
        br = br + (du + 2 * U) * np.abs(u) + U * np.abs(r)
    mean, dmean = 0.0, 0.0
    if norm == "layer":
        mean = r.mean(-1, keepdims=True)
        dmean = g * np.abs(r).mean(-1, keepdims=True) + br.max(-1, keepdims=True)
    d = r - mean
    rstd = 1.0 / np.sqrt(np.mean(d * d, -1, keepdims=True) + eps)
    n = d * rstd
    dd = br + dmean + U * np.abs(d)
    # the deviations' own errors move the variance by at most twice their largest, relative to the deviation
    bn = dd * rstd + np.abs(n) * (g / 2 + 6 * U + dd.max(-1, keepdims=True) * rstd)
    k = np.ones_like(n)
    if weight is not None:
        k = k * np.asarray(weight, np.float64)
    if scale is not None:
        k = k * (1.0 + _rows(scale, B, S))
    y = n * k
    by = (bn + 4 * U * np.abs(n)) * np.abs(k)
    if weight is not None and scale is not None:
        by = by + U * np.abs(n * np.asarray(weight, np.float64))  # 1 + scale, where it nearly cancels
    elif scale is not None:
        by = by + U * np.abs(n)
    if shift is not None:
        y = y + _rows(shift, B, S)
        by = by + U * np.abs(y)
    return r, y, br, by


# ---------------------------------------------------------------------------------------
# blocks of 32 four-bit values
# ---------------------------------------------------------------------------------------

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_quantize(x):
    """x [M, K] -> (codes [M, K / 2], scales [ceil(K / 256), M, 8]) uint8."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    v = x.reshape(M, K // 32, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(v).max(-1)
    bad = ~np.isfinite(top)
    frac, e = np.frexp(np.where(bad | (top == 0), 1.0, top))  # frac in [1/2, 1)
    e = np.where(top == 0, -127, np.maximum(e - 3 + (frac >= 0.875), -127))
    mag = np.where(bad[..., None], 0.0, np.abs(v)) / np.exp2(e.astype(np.float64))[..., None]
    # nearest code: the number of midpoints below, where a midpoint itself goes to the even code
    mid = (GRID[1:] + GRID[:-1]) / 2
    code = np.zeros(mag.shape, np.int64)
    for i, m in enumerate(mid):
        code += (mag > m) | ((mag == m) & (i % 2 == 1))
    code |= np.where(np.signbit(v), 8, 0)
    code = code.reshape(M, K)
    slabs = -(-K // 256)
    scales = np.full((M, slabs * 8), 127, np.int64)
    scales[:, : K // 32] = np.where(bad, 255, e + 127)
    scales = scales.reshape(M, slabs, 8).transpose(1, 0, 2)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8), np.ascontiguousarray(scales.astype(np.uint8))


def mxfp4_values(codes, scales):
    """The numbers that codes and scales stand for, [M, K]."""
    codes = np.asarray(codes, np.int64)
    M, K = codes.shape[0], 2 * codes.shape[1]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(M, K)
    v = np.where(c & 8, -GRID[c & 7], GRID[c & 7])
    e = np.asarray(scales, np.int64).transpose(1, 0, 2).reshape(M, -1)[:, : K // 32]
    p = np.where(e == 255, np.nan, np.exp2(e - 127.0))
    return (v.reshape(M, K // 32, 32) * p[..., None]).reshape(M, K)


def gelu_tanh(z):
    return 0.5 * z * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (z + 0.044715 * z ** 3)))


def mxfp4_linear(a, w, bias=None, act: bool = False):
    """a [M, K], w [N, K] (values) -> (act(a w^T + bias), bound of fp32 accumulation).

    The products of 8 neighbours, which lie in one block, are multiples of 1/4 up to 36 of one power of two
    and add without error; K / 8 such sums, the bias and what stands at the sum's start join the
    accumulator with at most 2 U (a truncation) of what the sum's terms amount to.  The activation's slope
    is under 1.13; its own arithmetic, a handful of operations and the exponential's argument, of up to 17
    in size where the result matters, is within 32 U |z|."""
    a, w = np.asarray(a, np.float64), np.asarray(w, np.float64)
    z = a @ w.T
    size = np.abs(a) @ np.abs(w).T
    if bias is not None:
        z = z + np.asarray(bias, np.float64)
        size = size + np.abs(np.asarray(bias, np.float64))
    bound = (a.shape[1] / 8 + 2) * 2 * U * size
    if act:
        return gelu_tanh(z), 1.13 * bound + 32 * U * np.abs(z)
    return z, bound
