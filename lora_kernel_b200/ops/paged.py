"""Page-scaled 8-bit KV cache: append, read-back, attention and page copies.

The cache of a layer is k_cache / v_cache [pages * page, Hkv, Dh] of
float8_e4m3fn or int8 codes and k_scale / v_scale [pages, Hkv] fp32, one
power-of-two scale per (page, KV head): the smallest that holds the page's
largest value.  Token t of a sequence lies at slot
table[t // page] * page + t % page, as in the cache with a scale per token.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .._ext import C, require_device, status

PAGE_KV = {"fp8_page": torch.float8_e4m3fn, "int8_page": torch.int8}


def new_page_cache(layers: int, num_pages: int, page: int, Hkv: int, Dh: int, kv_dtype: str = "fp8_page", device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of `layers` layers."""
    k = torch.zeros(layers, num_pages * page, Hkv, Dh, dtype=PAGE_KV[kv_dtype], device=device)
    ks = torch.zeros(layers, num_pages, Hkv, dtype=torch.float32, device=device)
    return k, torch.zeros_like(k), ks, torch.zeros_like(ks)


def page_append(qkv: torch.Tensor, Hq: int, Hkv: int, Dh: int, slots: torch.Tensor, k_cache, v_cache, k_scale,
                v_scale, page: int) -> None:
    """Write the keys and values of qkv [T, (Hq + 2 Hkv) * Dh] (bf16, after RoPE) to
    slots [T] (int32, negative = skip).

    A row at offset 0 of a page starts it afresh; any other row joins the rows
    before its offset, whose codes are moved to the page's new scale when that
    grows.  Rows of one page within a call are consecutive, in ascending order
    and without gaps.  Infinite values are stored as the largest code, NaN as 0."""
    require_device(qkv)
    C().page_append(qkv, Hq, Hkv, Dh, slots, k_cache, v_cache, k_scale, v_scale, page, status(qkv.device))


def page_gather(k_cache, v_cache, k_scale, v_scale, slots: torch.Tensor, Hkv: int, Dh: int, page: int,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The cached keys and values at `slots` (int32 [n]) as bf16 rows [n, 2 * Hkv * Dh]
    (exact: a code times a power of two), keys first."""
    require_device(k_cache)
    return C().page_gather(k_cache, v_cache, k_scale, v_scale, slots, Hkv, Dh, page, out, status(k_cache.device))


def page_attention(q: torch.Tensor, k_cache, v_cache, k_scale, v_scale, block_tables: torch.Tensor,
                   ctx_lens: torch.Tensor, page: int, Hq: int, Hkv: int, Dh: int, *, q_len: int = 1, max_ctx: int = 0,
                   scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [n * q_len, Hq * Dh] (bf16, after RoPE): the newest q_len tokens of each of n
    sequences, already appended -> out of the same shape.

    block_tables int32 [n, pages], ctx_lens int32 [n] (the q_len tokens
    included; 0 = unused row, which gives zeros).  Query j attends to positions
    0 .. ctx - q_len + j; the codes there are page_append's, which are finite
    (what lies in a page beyond a context is never read).  max_ctx: the longest length, where the host knows
    it (0: the tables' width); it only guides how the work is split."""
    require_device(q)
    return C().page_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, ctx_lens, page, Hq, Hkv, Dh, q_len,
                              max_ctx, 1.0 / math.sqrt(Dh) if scale is None else scale, out, status(q.device))


def copy_pages(caches: Sequence[torch.Tensor], moves: Union[torch.Tensor, List[Tuple[int, int]]], num_pages: int) -> None:
    """Copy pages in every layer of every tensor of a cache, in one launch.

    caches: contiguous tensors [layers, num_pages * rows, ...] (any type; codes
    and scales together).  moves: (source, destination) page ids, as a list or
    an int32 device tensor [n, 2].  No destination may appear twice or be a
    source: a list is checked, a tensor is taken at its word."""
    require_device(caches[0])
    if not isinstance(moves, torch.Tensor):
        dst = {d for _, d in moves}
        if len(dst) != len(moves) or any(s in dst for s, _ in moves):
            raise ValueError("copy_pages: a destination is named twice or is another move's source")
        if any(not 0 <= x < num_pages for m in moves for x in m):
            raise ValueError("copy_pages: page id out of range")
        moves = torch.tensor(moves, dtype=torch.int32).reshape(-1, 2).to(caches[0].device)
    C().copy_pages(list(caches), moves, num_pages, status(caches[0].device))
