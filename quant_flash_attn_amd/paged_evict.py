"""Eviction from a paged INT8 cache by accumulated attention weight.

    o, lse = quant_flash_attn_paged(q, cache, page_table, starts, sm_scale=sm_scale, return_lse=True)
    weights = paged_attention_weights(q, cache, lse, page_table, starts, sm_scale=sm_scale, weights=weights, out=weights)   # every step
    kept, weights, lengths = paged_cache_evict(cache, page_table, lengths, weights, keep, new_page_table, last=256)         # now and then

A slot is a place of a sequence in the cache: until a first eviction its position.  Behind an eviction every key head holds other tokens, in
order, and the next token goes to slot lengths[b] while its position goes on: rotate its query and key with norm_rope_pair (positions of
their own) and append the key as it is.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib


def paged_attention_weights(q: torch.Tensor, cache, lse: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                            counts: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
                            weights: Optional[torch.Tensor] = None, decay: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decay * weights (zeros if not given) and the attention weight that every key got from a call of quant_flash_attn_paged with the same
    arguments, which gave `lse` [B,H,N]: its softmax's probabilities, summed over the call's tokens and the query heads that share a key
    head.  fp32 [B,heads,S], S = pages of a sequence * page_size: of every slot; what no row sees gets nothing.

    out: where it goes (contiguous; it may be `weights`), in place of a new tensor.  Sums are made in a fixed order.  A query row that is
    not finite leaves its key head's weights not finite.
    """
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else float(sm_scale)
    return _lib.host().paged_weights(q, tuple(cache), lse, page_table, starts, counts, bool(causal), sm, weights, float(decay), out)


def paged_cache_evict(cache, page_table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, keep: int, new_page_table: torch.Tensor,
                      first: int = 0, last: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of every sequence's lengths[b] slots each key head keeps min(lengths[b], keep): the `first` first and `last` last ones always
    (first + last <= keep), of the others the heaviest (weights [B,heads,S] fp32; ties: the lowest slot; NaN below all numbers).

    Their rows move, in order, to the pages of new_page_table int32 [B, at least keep / page_size], which must stand in no page table of
    the call elsewhere; the old pages stay as they are, so they may be shared with other sequences, and are free afterwards.  A sequence of
    length 0 is passed over; a -1 in new_page_table skips that page's rows.
    Returns the kept slots, int32 [B,heads,keep], ascending, -1 behind; their weights [B,heads,new S], zeros behind; the new lengths [B].
    """
    return _lib.host().paged_evict(tuple(cache), page_table, lengths, weights, int(keep), new_page_table, int(first), int(last))
