"""A paged INT8 cache of keys and values, and attention on it, for batches of sequences of different length.

The rows are quantized per token as asymmetric_quant_per_token does it, and lie in pages of a power of two of rows, 16 at least:
position p of sequence b is row p % page_size of page page_table[b, p // page_size].  Lengths and page tables stay on the
device (int32): nothing here waits for them, and a captured graph follows them as they change.

    cache = make_paged_cache(pages, heads, page_size, head_dim)
    paged_cache_append(cache, k, v, page_table, starts, cos=cos, sin=sin)            # the new tokens' keys and values
    o = quant_flash_attn_paged(q, cache, page_table, starts, sm_scale=sm_scale)      # their queries on all of them

`starts` [B] is the position of every sequence's first new token, the same for both calls; `counts` [B] (optional) how many of the
call's N tokens a sequence brings (the others are padding behind them).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib


class PagedCache(NamedTuple):
    k_codes: torch.Tensor       # int8 [pages, heads, page_size, head_dim]
    k_scale: torch.Tensor       # [pages, heads, page_size, 1], fp16, bf16 or fp32
    k_zero_point: torch.Tensor  # int8 [pages, heads, page_size, 1]
    v_codes: torch.Tensor
    v_scale: torch.Tensor
    v_zero_point: torch.Tensor


def make_paged_cache(pages: int, heads: int, page_size: int, head_dim: int, scale_dtype: torch.dtype = torch.float16,
                     device="cuda") -> PagedCache:
    """An empty cache (fp16 scales by default, as asymmetric_quant_per_token returns them)."""
    def side():
        shape = (pages, heads, page_size)
        return (torch.zeros(*shape, head_dim, dtype=torch.int8, device=device),
                torch.zeros(*shape, 1, dtype=scale_dtype, device=device), torch.zeros(*shape, 1, dtype=torch.int8, device=device))
    return PagedCache(*side(), *side())


def paged_cache_append(cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                       counts: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                       cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       interleaved: bool = False) -> None:
    """Quantizes k and v [B,heads,N,D] (fp16, bf16 or fp32) into the cache, in place and in one launch: token n < counts[b] goes to
    position starts[b] + n of its sequence.

    The keys are normed (k_weight, eps) and rotated by their position (cos, sin, interleaved) on the way, as norm_rope does it, without
    a rounding in between.  A token has no place, and neither its keys nor its values are written, where its position is negative, past
    the page table or past the table of angles, or its page is none of the cache's (so a -1 in the page table skips).  A page that is
    written may stand only once in the call's page table (pages that sequences share may be read by all of them).  No gradient flows
    through a cache.
    """
    _lib.host().paged_append(tuple(cache), k, v, page_table, starts, counts, k_weight, cos, sin, float(eps), bool(interleaved))


def paged_cache_read(cache, page_table: torch.Tensor, starts: torch.Tensor, N: int, counts: Optional[torch.Tensor] = None,
                     dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [B,heads,N,D] of positions starts[b] + n as what their codes stand for, (code - zero point) * scale, rounded to
    dtype; zeros from counts[b] on and for positions without a page."""
    return _lib.host().paged_read(tuple(cache), page_table, starts, int(N), counts, dtype)


def quant_flash_attn_paged(q: torch.Tensor, cache, page_table: torch.Tensor, starts: torch.Tensor,
                           counts: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
                           prefix_len: int = 0, return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the tokens at the end of every sequence, q [B,H,N,D], on its pages; H a multiple of the cache's heads (query head h
    reads key head h // (H // heads)).  O [B,H,N,D] of q's type.  The arithmetic is quant_flash_attn_quantized_kv's for short query
    blocks: queries quantized per token inside, INT8 scores, V as its exact codes.  No gradient.

    Token n < counts[b] is at position starts[b] + n and sees the keys up to itself (causal False: all starts[b] + counts[b]); its own
    key has to be in the cache.  Padding tokens, and tokens that see no key, get zeros.
    prefix_len: the first prefix_len positions hold the same rows for all sequences, as a common system prompt (in pages that stand in all
        their page tables, or in copies).  Where that pays they are read once for all of them, from sequence 0's pages: its row of the page table has
        to hold them also if it brings no token to this call.
    sm_scale: 1 / sqrt(D) if not given.
    return_lse: also the log-sum-exp of every row's scaled scores, fp32 [B,H,N] (-inf where a row sees no key); O has the same bits.
    The keys are dealt to workgroups evenly over the whole batch: the last bits of a sequence's O depend on the other sequences'
    lengths; the same call gives the same bits.
    """
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else float(sm_scale)
    call = _lib.host().paged_attn_lse if return_lse else _lib.host().paged_attn
    return call(q, tuple(cache), page_table, starts, counts, bool(causal), sm, int(prefix_len))
