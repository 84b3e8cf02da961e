"""The paged e4m3 cache of keys and values and the attention over it, in 64 bits (test infrastructure only).

Written from the definitions, token by token.  Functions that a kernel's 32-bit arithmetic follows within
rounding return the bound of that rounding beside the result.
"""
from __future__ import annotations

import math

import numpy as np

from .dit_block import rotate
from .numerics import e4m3_decode, e4m3_encode

E_MIN, E_MAX = -32, 63


def exponent(amax: float) -> int:
    """The smallest e in [-32, 63] with amax <= 448 * 2^e."""
    e = E_MIN
    while e < E_MAX and amax > math.ldexp(448.0, e):
        e += 1
    return e


def round_codes(x, e: int):
    """The e4m3 codes nearest to x * 2^-e (fp64), ties to even, 448 at the most; NaN as 0."""
    y = np.clip(np.nan_to_num(np.ldexp(np.asarray(x, np.float64), -e), nan=0.0, posinf=448.0, neginf=-448.0), -448, 448)
    a = np.abs(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 1e-300))), -6.0) - 3.0)
    return e4m3_encode(np.copysign(np.minimum(np.rint(a / step) * step, 448.0), y).astype(np.float32))


class Pool:
    """Codes [pages, H, page, D] and scale bytes [pages, H] of keys (0) and values (1), as numpy arrays."""

    def __init__(self, codes, scales):
        self.codes, self.scales = [np.array(c) for c in codes], [np.array(s) for s in scales]
        self.page = self.codes[0].shape[2]

    def copy(self):
        return Pool(self.codes, self.scales)

    def at(self, table, b, t):
        """(page, slot) of sequence b's token t, or None."""
        if t < 0 or t // self.page >= table.shape[1]:
            return None
        p = int(table[b, t // self.page])
        return (p, t % self.page) if 0 <= p < self.codes[0].shape[0] else None

    def value(self, which, p, h, slot):
        return np.ldexp(e4m3_decode(self.codes[which][p, h, slot]).astype(np.float64), int(self.scales[which][p, h]) - 127)


def append(pool: Pool, table, starts, k, v, counts=None, turns=None, weight=None, eps=1e-6, interleaved=True):
    """Appends k, v [B, H, S, D] to `pool`, page by page.  Returns the unrounded keys and values [B, H, S, D] and the
    bound of what 32-bit arithmetic may add to the keys."""
    B, H, S, D = k.shape
    if turns is None:
        turns = np.zeros((S, 0, 2))
    key, bound = rotate(k, turns, weight, eps, interleaved)
    new = [key, np.asarray(v, np.float64)]
    for b in range(B):
        n = S if counts is None else min(max(int(counts[b]), 0), S)
        start = int(starts[b])
        pages = {}
        for s in range(n):
            at = pool.at(table, b, start + s)
            if at:
                pages.setdefault(at[0], []).append((s, at[1]))
        for p, tokens in pages.items():
            old = tokens[0][1] if tokens[0][0] == 0 else 0  # slots held by tokens before `start`
            for h in range(H):
                for which in range(2):
                    x = np.stack([new[which][b, h, s] for s, _ in tokens])
                    a = np.abs(x[np.isfinite(x)])
                    e = exponent(a.max() if a.size else 0.0)
                    held = int(pool.scales[which][p, h]) - 127
                    if old:
                        e = max(e, held)
                        if e > held:
                            c = pool.codes[which][p, h, :old]
                            again = round_codes(e4m3_decode(c).astype(np.float64), e - held)
                            pool.codes[which][p, h, :old] = np.where(c & 0x7F == 0x7F, c, again)
                    for (s, slot), row in zip(tokens, x):
                        pool.codes[which][p, h, slot] = round_codes(row, e)
                    pool.scales[which][p, h] = e + 127
                for s, slot in tokens:
                    if np.isnan(new[0][b, h, s]).any() or np.isnan(new[1][b, h, s]).any():
                        pool.codes[0][p, h, slot, 0] |= 0x7F
    return new[0], new[1], bound


def read(pool: Pool, table, starts, tokens: int, lengths=None):
    """(k, v) [B, H, tokens, D], zeros where there is nothing."""
    B, H, D = len(starts), pool.codes[0].shape[1], pool.codes[0].shape[3]
    out = np.zeros((2, B, H, tokens, D))
    for b in range(B):
        for t in range(tokens):
            at = pool.at(table, b, int(starts[b]) + t)
            if at and (lengths is None or int(starts[b]) + t < int(lengths[b])):
                for h in range(H):
                    for which in range(2):
                        out[which, b, h, t] = pool.value(which, at[0], h, at[1])
    return out


def attend(q, k, v, there, lengths, scale: float, causal: bool = False, q_lengths=None):
    """q [B, H, S, D] over the tokens k, v [B, Hk, T, D] of each sequence's table; there [B, T]: tokens that have a
    page.  Returns (o, a): the outputs, and sum p |v| / sum p, which bounds of the rounding are relative to."""
    B, H, S, D = q.shape
    T, G = k.shape[2], H // k.shape[1]
    o, a = np.zeros((B, H, S, D)), np.zeros((B, H, S, D))
    for b in range(B):
        length = int(lengths[b])  # (past the table's end there are no tokens, but the diagonal counts from it)
        n = S if q_lengths is None else min(max(int(q_lengths[b]), 0), S)
        for i in range(n):
            seen = there[b] & (np.arange(T) < (length - n + i + 1 if causal else length))
            if not seen.any():
                continue
            for h in range(H):
                kk, vv = k[b, h // G][seen], v[b, h // G][seen]
                x = kk @ q[b, h, i] * scale
                p = np.exp(x - x.max())
                o[b, h, i], a[b, h, i] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
    return o, a


def attend_small(q, k, v, e, lengths, scale: float, causal: bool = False):
    """As `attend`, all tokens there; e [B, Hk, T]: the exponents of the values' pages.  Returns (o, a, small).

    The kernels round p 2^e to fp16 with the row's largest so far at 2^7 or above: half a step of the smallest numbers,
    2^-25, is 2^-32 of that largest.  `small` is this for each key, times the value's code, over sum p."""
    B, H, S, D = q.shape
    T, G = k.shape[2], H // k.shape[1]
    o, a, small = np.zeros((3, B, H, S, D))
    for b in range(B):
        for h in range(H):
            kk, vv, ee = k[b, h // G], v[b, h // G], np.exp2(e[b, h // G].astype(np.float64))
            codes = np.abs(vv) / ee[:, None]
            x = q[b, h] @ kk.T * scale
            seen = np.arange(T) < (lengths[b] - S + np.arange(S)[:, None] + 1 if causal else lengths[b])
            x = np.where(seen, x, -np.inf)
            p = np.exp(x - x.max(-1, keepdims=True))
            total = p.sum(-1, keepdims=True)
            o[b, h], a[b, h] = p @ vv / total, p @ np.abs(vv) / total
            small[b, h] = 2.0 ** -32 * (p * ee).max(-1, keepdims=True) * (seen @ codes) / total
    return o, a, small
