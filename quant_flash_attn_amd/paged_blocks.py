"""Attention on a long paged INT8 cache that reads only some of its blocks: those that a cheap score selects for each token.

A block is a page.  Beside the cache lie the bounds of every page's keys, and a token's queries are scored against those in place of
the keys themselves:

    bounds = make_page_bounds(cache)
    paged_cache_append(cache, k, v, page_table, starts, cos=cos, sin=sin)                        # as ever
    paged_bounds_update(bounds, cache, page_table, starts, N)                                    # of the pages that this touched
    blocks = paged_select_blocks(q, cache, bounds, page_table, starts, keep=64)                  # 64 blocks for every token and key head
    o = quant_flash_attn_paged_blocks(q, cache, page_table, starts, blocks, sm_scale=sm_scale)

Lengths, page tables and lists stay on the device, and a captured graph follows them.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib


class PageBounds(NamedTuple):
    codes: torch.Tensor        # int8 [pages, heads, 2, head_dim]: the low and the high row
    scale: torch.Tensor        # fp32 [pages, heads, 2, 1]
    zero_point: torch.Tensor   # int16 [pages, heads, 2, 1]


def make_page_bounds(cache) -> PageBounds:
    """Room for the bounds of all pages of a cache (an empty one; paged_bounds_update fills them in)."""
    pages, heads, _, head_dim = cache[0].shape
    device = cache[0].device
    return PageBounds(torch.zeros(pages, heads, 2, head_dim, dtype=torch.int8, device=device),
                      torch.zeros(pages, heads, 2, 1, dtype=torch.float32, device=device),
                      torch.zeros(pages, heads, 2, 1, dtype=torch.int16, device=device))


def paged_bounds_update(bounds, cache, page_table: torch.Tensor, starts: torch.Tensor, N: int, counts: Optional[torch.Tensor] = None) -> None:
    """The bounds of the pages that positions starts[b] .. starts[b] + n - 1 lie in (n = N, or counts[b] of them), in place and in one launch:
    of every element the smallest and the largest key of the page's rows before starts[b] + n, the two rows quantized as asymmetric_quant_per_token
    does it, but with zero points of 16 bits: rows of one sign, which the least and the largest keys of a page often are, have theirs outside of 8.
    (Bounds whose zero points are int8 are taken too: their rows are quantized as tokens are, and of a row of one sign what lies
    further from zero than its span is cut, so that such bounds may fall short of their page's keys.)

    With the arguments of every paged_cache_append it keeps all bounds up to date (after paged_cache_evict: the new pages', from position 0
    on).  A page that is written may stand only once in the call's page table.
    """
    _lib.host().paged_bounds(tuple(bounds), tuple(cache), page_table, starts, int(N), counts)


def paged_select_blocks(q: torch.Tensor, cache, bounds, page_table: torch.Tensor, starts: torch.Tensor, keep: int,
                        counts: Optional[torch.Tensor] = None, first: int = 1, last: int = 1,
                        return_scores: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """For every token of q [B,H,N,D] (at position starts[b] + n) and key head the numbers of `keep` blocks up to its own: int32
    [B,heads,N,keep], ascending, -1 behind (all of them for padding tokens).

    Selected are the blocks whose keys may have the largest product with one of the query heads that share the key head: the score is
    the sum over elements of max(q low, q high), the query quantized per token, exact but for one rounding to fp32: what a key of the block may
    have at most, but for half a step of the bounds' codes.  Ties go to the
    lowest number; the `first` first and `last` last blocks that a token sees are always taken (first + last <= keep).
    return_scores: also the scores [B,heads,N,pages of a sequence], fp32, -inf for blocks that a token does not see or that have no page.
    """
    blocks, scores = _lib.host().paged_select(q, tuple(cache), tuple(bounds), page_table, starts, int(keep), counts, int(first), int(last),
                                              bool(return_scores))
    return (blocks, scores) if return_scores else blocks


def quant_flash_attn_paged_blocks(q: torch.Tensor, cache, page_table: torch.Tensor, starts: torch.Tensor, blocks: torch.Tensor,
                                  counts: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None) -> torch.Tensor:
    """quant_flash_attn_paged (causal) of every token on its own list of blocks, int32 [B,heads,N,keep]: O [B,H,N,D] of q's type, the same
    arithmetic (of fp32 queries without its 16-bit rounding of probabilities).  No gradient.

    A token sees the keys up to itself in the blocks of its list.  The order of a list does not matter, a block that stands in it twice
    counts twice, numbers outside the page table and blocks without a page are passed over.  Tokens that see no key, and padding, get zeros.
    """
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else float(sm_scale)
    return _lib.host().paged_blocks(q, tuple(cache), page_table, starts, blocks, counts, sm)
