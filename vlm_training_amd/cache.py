"""Serving with full attention: a paged cache of keys and values, and attention over it.

``KvCache``         one layer's pages, bf16 or 8-bit (e4m3 with a power of two for each row of each head).
``kv_cache_write``  puts the keys and values of new tokens on their requests' pages.
``kv_cache_read``   gives rows back, packed, as the operators of packed sequences take them.
``paged_attn``      the new tokens of each request - one, some drafted ones, a chunk of a prompt or all of it - over what the cache holds of it.

The reference trains only and keeps no cache; these are what its attention layers (models/qwen3_vl/model.py:230-278, models/qwen3_5/model.py:76-136) need to answer, as
``gated_delta_step`` and ``short_conv_step`` are for its linear-attention layers.  Host side in csrc/dsa_host_cache.cpp over the C ABI; there is no fallback path.

Every call takes ``page_table`` (N, P) int32: position p of request n lies on page ``page_table[n, p // page]``, at ``p % page``.  What lies on no page - a page number outside
the pool, -1 for one, or a position outside the table - is not written and reads as zero.  ``cu_seqlens`` (N+1,) are the offsets of the requests' new rows in the packed tensors (requests
without any are allowed, rows behind the last one give zeros), ``lengths`` (N,) the requests' lengths with their new rows.  Integers are int32, or int64, which costs a
conversion.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib


@dataclass
class KvCache:
    """The pages of one layer: ``k``, ``v`` (pages, kv heads, page, head_dim) bf16 or float8_e4m3fn, a page's rows contiguous (slices of a pool for all layers will do);
    ``page`` is 16, 32, 64, 128 or 256, ``head_dim`` a multiple of 8 (8-bit: 16) up to 256.

    An 8-bit cache has ``k_scale``, ``v_scale`` (pages, kv heads, page) float8_e8m0fnu: a value stands for itself times its row's power of two, the smallest one (from 2^-100 on) with
    which the row's largest value is at most 448.  That rounds a value by at most 2^-4 of itself, or 2^-10 of the power for values under 2^-6 of it, and what is stored is exact in
    bf16 (next to bf16's largest value it is 240 * 2^120 at the most, not 2^128).  A row with a value that is not finite is NaN as a whole."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, *, page: int = 64, dtype=torch.bfloat16, device="cuda"):
        """A cache of zeros; ``dtype`` torch.bfloat16 or torch.float8_e4m3fn."""
        if page not in (16, 32, 64, 128, 256):
            raise ValueError(f"a page holds 16, 32, 64, 128 or 256 rows, not {page}")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"a cache holds torch.bfloat16 or torch.float8_e4m3fn, not {dtype}")
        k, v = (torch.zeros(pages, heads, page, head_dim, dtype=torch.uint8 if dtype.itemsize == 1 else dtype, device=device).view(dtype) for _ in range(2))
        if dtype == torch.bfloat16:
            return cls(k, v)
        return cls(k, v, *(torch.zeros(pages, heads, page, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu) for _ in range(2)))

    def _parts(self):
        return self.k, self.v, self.k_scale, self.v_scale


@torch.compiler.disable
def kv_cache_write(cache: KvCache, k, v, page_table, cu_seqlens, lengths) -> None:
    """k, v (T, kv heads, head_dim) bf16 views: request n's rows ``cu_seqlens[n]`` to ``cu_seqlens[n + 1]`` become its last ones, positions ``lengths[n]`` minus their number on.

    The cache is updated in place.  Two rows for one place (a page in two requests' tables where both write, keys and values in the same memory) are written in no order; pages
    that are only read may be shared.  ``k`` and ``v`` may lie in the pools themselves (a page copied to another), but not where the call writes: what it then reads is one or
    the other.  No backward pass."""
    _lib.host().kv_cache_write(*cache._parts(), k, v, page_table, cu_seqlens, lengths)


@torch.compiler.disable
def kv_cache_read(cache: KvCache, page_table, cu_seqlens, rows: int, *, first=None):
    """Keys and values (rows, kv heads, head_dim) bf16: rows ``cu_seqlens[n]`` to ``cu_seqlens[n + 1]`` are request n's positions ``first[n]`` on (0 without ``first``).

    ``rows`` is the number of rows in all; those behind the last request give zeros.  What an 8-bit cache holds is exact in bf16.  No backward pass."""
    return tuple(_lib.host().kv_cache_read(*cache._parts(), page_table, cu_seqlens, int(rows), first))


@torch.compiler.disable
def paged_attn(q, cache: KvCache, page_table, cu_seqlens, lengths, *, max_new=None, max_length=None, softmax_scale=None, return_lse: bool = False):
    """q (T, q heads, head_dim) bf16 view -> (T, q heads, head_dim): causal attention of each request's new rows over its cached keys and values, their own (already
    written) ones among them; q head h reads kv head ``h // (q heads // kv heads)``, up to 16 to one.

    A row without any key - its request is shorter than its new rows - gives zeros; a key or value that a row does not attend never reaches it, not finite ones either; a
    NaN logit that it does attend makes it NaN.
    ``max_new`` and ``max_length``, where known, are upper bounds of the requests' new rows and lengths: with them fewer kernels are launched; results do not depend on them but for
    the order of sums.  ``softmax_scale`` defaults to ``head_dim ** -0.5``.  ``return_lse`` adds (q heads, T) fp32: the logarithm of each row's sum of exponentials, -inf
    for rows without a key.  Probabilities are rounded to bf16 for their product with the values; statistics and sums are fp32.  Sums are
    divided at the end, with weights of up to 2^8: values up to 2^89 never pass their range.  No backward pass."""
    out = _lib.host().paged_attn(q, *cache._parts(), page_table, cu_seqlens, lengths, max_new, max_length, softmax_scale, bool(return_lse))
    return tuple(out) if return_lse else out[0]
