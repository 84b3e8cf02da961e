"""A paged cache of keys and values in 8 bits, and attention over it (an extension; no counterpart in the
reference's files).

``fp8_attention`` quantizes all keys and values of a call at once: its scales need the whole sequence's
mean key and each channel's largest value.  A clip that is generated a few frames at a time, a prompt
that is read and continued, or a text context that every denoising step attends to keep theirs in an
``FP8KVCache`` instead: e4m3 codes in pages of a few tokens, with a power-of-two scale for each page
and head, so that a token can be added without a look at the others.  ``append_kv`` norms, turns and
quantizes new keys and values into the pages, ``cached_attention`` attends to them, and ``read_kv``
gives the values back.

Pages belong to whoever hands them out: a call names each sequence's pages in a ``page_table``
[B, W] int32, token t of sequence b in page ``page_table[b, t // page_size]``.  An entry that is no page
of the cache (-1) stands for none.  Dropping the pages of a clip's oldest frames from the table ends the
attention to them; two sequences may share the pages of a common beginning, as long as neither
appends to them.
"""
from __future__ import annotations

import math

import torch

from .. import ops

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class FP8KVCache:
    """``pages`` pages of ``page_size`` tokens with ``heads`` key heads of ``head_dim`` channels.

    k, v: e4m3 codes [pages, heads, page_size, head_dim]; k_scale, v_scale: uint8 [pages, heads], the
    exponent + 127 of the power of two that the page's codes are times.
    """

    def __init__(self, pages: int, heads: int, head_dim: int, page_size: int = 64,
                 device: torch.device | str = "cuda") -> None:
        codes = [torch.zeros((pages, heads, page_size, head_dim), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.full((pages, heads), 127, dtype=torch.uint8, device=device) for _ in range(2)]
        self._set(*codes, *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> FP8KVCache:
        """A cache on these tensors themselves (codes as e4m3 or their bytes).  Scale bytes of pages in use are 95
        to 190, as ``append_kv`` writes them, and their values hold no NaN."""
        cache = cls.__new__(cls)
        cache._set(k, v, k_scale, v_scale)
        return cache

    def _set(self, k, v, k_scale, v_scale):
        for t in (k, v):
            if t.dtype not in (torch.uint8, ops.E4M3) or t.dim() != 4 or t.shape != k.shape or not t.is_contiguous():
                raise ValueError("FP8KVCache: k and v must be contiguous e4m3 codes [pages, heads, page_size, head_dim], "
                                 f"got {t.dtype} {tuple(t.shape)}")
        for t in (k_scale, v_scale):
            if t.dtype != torch.uint8 or t.shape != k.shape[:2] or not t.is_contiguous():
                raise ValueError(f"FP8KVCache: scales must be contiguous uint8 {tuple(k.shape[:2])}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        if k.shape[2] not in PAGE_SIZES:
            raise ValueError(f"FP8KVCache: page_size must be one of {PAGE_SIZES}, got {k.shape[2]}")
        if k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"FP8KVCache: head_dim must be one of {HEAD_DIMS}, got {k.shape[3]}")
        if not k.device == v.device == k_scale.device == v_scale.device:
            raise ValueError("FP8KVCache: all tensors must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k.view(ops.E4M3), v.view(ops.E4M3), k_scale, v_scale

    pages = property(lambda self: self.k.shape[0])
    heads = property(lambda self: self.k.shape[1])
    page_size = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])
    device = property(lambda self: self.k.device)

    def tensors(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.k, self.v, self.k_scale, self.v_scale


def append_kv(cache: FP8KVCache, page_table: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
              counts: torch.Tensor | None = None, table: torch.Tensor | None = None,
              k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = True) -> None:
    """Writes k, v [B, Hk, S, D] (bf16, fp16 or fp32, any strides) into the cache, as tokens
    ``starts[b]`` ... of sequence b; with ``counts`` [B] only the first counts[b] of each.

    starts, counts: int32 [B].  ``table`` [S, P, 2] or [B, S, P, 2] turns the keys and ``k_weight`` [D]
    norms them per head before, as ``rotate_qk`` does, without its rounding between.  Tokens from
    starts[b] on count as not there before: a chunk can be appended again at the same place (a denoising
    step later), or a sequence cut.  A page's scale is the smallest power of two that holds what is
    appended, or the one it has where that is larger and tokens before starts[b] use it; where it
    grows those are rounded again.  Exponents go from -32 to 63: values from 1.5e-12 to 4e21 in size.

    An infinity is held as the largest number.  A NaN in a token's key or value makes the rows that attend
    to that token (and head) NaN, and no others.  Tokens behind the page table's last entry, or where
    it names no page, are dropped.  A page may not be written to through two entries of the table.
    """
    ops.kv_append(*cache.tensors(), page_table, starts, k, v, counts, table, k_weight, float(eps), bool(interleaved))


def cached_attention(q: torch.Tensor, cache: FP8KVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                     scale: float | None = None, causal: bool = False,
                     q_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of q [B, H, S, D] (bf16 or fp16) over the first ``lengths[b]`` cached tokens of
    each sequence; [B, H, S, D] in q's dtype and order of dimensions.

    H is a multiple of the cache's heads, and head h attends to key head h // (H / Hk).  With ``q_lengths``
    [B] only the first q_lengths[b] queries of a sequence are there, and the others' rows are 0.
    ``causal``: the queries are the sequence's last tokens, already appended, and each sees the keys up to its
    own (also where ``lengths`` is past the table, and the last tokens were dropped; without it all see all: a
    frame's tokens among each other, or text).  A row that sees no key is 0.  lengths, q_lengths: int32 [B].  scale
    defaults to 1 / sqrt(D).

    Codes are used as they are, q and the probabilities in fp16 under scales of their own, and scores and sums are
    fp32 (a row with a score past 3.4e38 in size may be NaN).  The same call gives the same bits; a row's last bit may
    differ between calls of different shapes.
    """
    return ops.kv_attend(q, *cache.tensors(), page_table, lengths, q_lengths, bool(causal),
                         1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale))


def read_kv(cache: FP8KVCache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int, *,
            lengths: torch.Tensor | None = None,
            dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of ``tokens`` tokens of each sequence from ``starts[b]`` (int32) on, [B, Hk, tokens, D]:
    exact in bf16 and fp32, rounded in fp16; 0 from token ``lengths[b]`` on and where there is no page."""
    return ops.kv_read(*cache.tensors(), page_table, starts, int(tokens), lengths, dtype)
