"""An 8-bit paged key/value cache: QuantizedKVCache, append_kv, attend_kv and
dequantize_kv (include/cublade_kv.h). No counterpart in the reference.

A served model's keys and values as INT8 or FP8 E4M3 codes, with one fp32 scale
for each page (a block of page_size tokens of one sequence) and kv head, in the
formats of quantize_tensor. A step of a model's layer is

    q = append_kv(cache, k, v, page_table, lengths, rope=(cos, sin), q=q)
    o = attend_kv(q, cache, page_table, lengths)

with the same page_table [batch, max_pages] and lengths [batch] (int32; the
tokens of every sequence with the new ones) in both calls. New tokens of all
sequences are packed along dimension 0: one each, or cu [batch + 1] gives where
each sequence's begin.
"""
from __future__ import annotations

import torch

from cublade_amd.bindings.hip.kv_cache import (STORE_CODE, kv_append, kv_attend, kv_cache_view,
                                               kv_dequantize)


class QuantizedKVCache:
    """The pool of pages.

    k: codes [num_pages, kv_heads, page_size, head_dim]; v: codes, transposed,
    [num_pages, kv_heads, head_dim, page_size]; k_scale, v_scale: float32
    [num_pages, kv_heads], not negative. All contiguous, on one device. head_dim: a multiple
    of 16 up to 256; page_size: 16, 32, 64, 128 or 256. The tensors are fixed:
    write into them, or make another cache.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "_view")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor):
        object.__setattr__(self, "_view", kv_cache_view(k, v, k_scale, v_scale))
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            object.__setattr__(self, name, t)

    def __setattr__(self, name, value):
        raise AttributeError(f"QuantizedKVCache.{name} is fixed")

    def __delattr__(self, name):
        raise AttributeError(f"QuantizedKVCache.{name} is fixed")

    def __reduce__(self):
        # pickle and deepcopy make the view of the new tensors anew
        return QuantizedKVCache, (self.k, self.v, self.k_scale, self.v_scale)

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
              dtype: torch.dtype = torch.int8, device="cuda") -> "QuantizedKVCache":
        """A pool of zeroed pages."""
        if dtype not in STORE_CODE:
            raise ValueError(f"QuantizedKVCache: dtype must be torch.int8 or torch.float8_e4m3fn, "
                             f"got {dtype}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"QuantizedKVCache: the cache must be on CUDA, got device={device}")
        shape = (num_pages, kv_heads, page_size, head_dim)
        k = torch.zeros(shape, dtype=torch.uint8, device=dev).view(dtype)
        v = torch.zeros((num_pages, kv_heads, head_dim, page_size), dtype=torch.uint8,
                        device=dev).view(dtype)
        scales = torch.zeros((2, num_pages, kv_heads), dtype=torch.float32, device=dev)
        return cls(k, v, scales[0], scales[1])

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def num_pages(self) -> int:
        return self._view.num_pages

    @property
    def kv_heads(self) -> int:
        return self._view.kv_heads

    @property
    def head_dim(self) -> int:
        return self._view.head_dim

    @property
    def page_size(self) -> int:
        return self._view.page_size

    def __repr__(self) -> str:
        return (f"QuantizedKVCache(num_pages={self.num_pages}, kv_heads={self.kv_heads}, "
                f"head_dim={self.head_dim}, page_size={self.page_size}, dtype={self.dtype}, "
                f"device={self.device})")


def append_kv(
    cache: QuantizedKVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    cu_new: torch.Tensor | None = None,
    rope: tuple[torch.Tensor, torch.Tensor] | None = None,
    interleaved: bool = False,
    positions: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Append new keys and values to the cache, in place; one launch.

    Args:
        k, v: [tokens, kv_heads, head_dim], fp16 or bf16, any strides (read in
            place where the last dimension is contiguous and the others are
            multiples of 8 elements, as in a fused projection's output).
        page_table: int32 [batch, max_pages], the page ids of every sequence.
        lengths: int32 [batch], tokens of every sequence with the new ones.
        cu_new: int32 [batch + 1], not decreasing: where each sequence's new
            tokens begin among `tokens`, and where the last one's end; None:
            one new token each. Tokens in front of them and behind them (a batch
            padded to a fixed size) are not appended; their queries are NaN
            where they would be rotated, unless `positions` are given.
        rope: (cos, sin), float32 [rows, rot_dim / 2]: k and q are rotated by
            the row of the token's position, dimensions i and i + rot_dim / 2
            as a pair (2 i and 2 i + 1 if `interleaved`), dimensions from
            rot_dim on as they are. The cache holds rotated keys.
        positions: int64 [tokens], the row for each token in place of its index
            in its sequence.
        q: [tokens, q_heads, head_dim]; the result is q rotated.

    A page's scale follows from the tokens it gets first; it grows by powers of
    two when later tokens need it, and the page's earlier codes are lowered
    with it. Sequences must not share a page that a call writes. A token whose
    page id is outside the pool, or whose position is outside the table, is
    dropped (attending to such a page gives NaN); one without a row in the
    rotation tables makes its query, and whatever attends to its page, NaN.
    Neither the cache nor the result carries a gradient.
    """
    return kv_append(cache._view, cache.k.device, k, v, page_table, lengths, cu_new, rope,
                     interleaved, positions, q)


def attend_kv(
    q: torch.Tensor,
    cache: QuantizedKVCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    cu_q: torch.Tensor | None = None,
    scale: float | None = None,
    causal: bool = True,
    window: int | None = None,
    max_length: int | None = None,
    return_lse: bool = False,
):
    """Attention of new tokens' queries over their sequences' cached tokens.

    Args:
        q: [tokens, q_heads, head_dim], fp16 or bf16; q_heads a multiple of
            kv_heads (query head h reads kv head h // (q_heads // kv_heads)).
        page_table, lengths: as given to append_kv; cu_q: as its cu_new. The n
            queries of a sequence are its last n tokens. A query outside cu_q
            sees no token.
        scale: of the scores, 1 / sqrt(head_dim) by default.
        causal: a query sees its own token and earlier ones; else all of its
            sequence's.
        window: with causal, only the last `window` of those.
        max_length: an upper bound of lengths known to the host. Only how the
            work is cut depends on it; without it, the page table's width.
        return_lse: also return the log-sum-exp of the scores, float32
            [tokens, q_heads].

    Returns [tokens, q_heads, head_dim] in q's dtype (and the log-sum-exp). A
    query that sees no token gives zeros, and -infinity (one whose scores are all
    -infinity NaN, and -infinity). The result carries no gradient.

    Scores, softmax statistics and sums are fp32, and the codes exact; fewer bits
    are kept in two places. Probabilities are rounded to fp16 for their product
    with the values (the sum that divides it takes them before that): 2^-11 of
    each, and 2^-25 of the largest product of a probability and its page's value
    scale, so a page's values lose bits where they are far below another page's.
    bf16 queries are fp16 numbers times a power of two for each row, so elements
    below 2^-25 of their row's largest vanish. Where value scales that a query
    sees lie more than 2^100 apart (fp16 values never do; scales below 2^-64
    count as 2^-64), the pages of the smallest ones may be left out of the sum.
    """
    return kv_attend(cache._view, cache.k.device, q, page_table, lengths, cu_q, scale, causal,
                     window, max_length, return_lse)


def dequantize_kv(cache: QuantizedKVCache, pages: torch.Tensor,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) of the given pages (int32 [n]) as [n, kv_heads, page_size,
    head_dim] in fp16 or bf16: (float(code) * scale).to(dtype), token-major
    both. A page id outside the pool reads as NaN."""
    return kv_dequantize(cache._view, cache.k.device, pages, dtype)
