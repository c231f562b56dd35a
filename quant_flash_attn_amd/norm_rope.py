"""RMSNorm of every head's queries and keys and the position rotation, in one pass, in front of the attention entry points.

The reference's operators take queries and keys as they come (quant_flash_attn.py:178); a model norms and rotates them first.
Both entry points are differentiable (a HIP kernel of its own, csrc/qfa_norm_rope.hip; no forward-mode and no second derivative).
An input is kept for its gradient only where it has a weight; what is rotated alone may change before the gradient is taken.
As with every torch backward pass, one that is captured into a HIP graph needs that no eager graph of the same leaves is alive then.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def rope_table(positions: int, rotated: int, base: float = 10000.0, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of p * base^(-2i / rotated), fp32 [positions, rotated / 2], from angles in 64 bits: made once, kept by the caller."""
    rate = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return angle.cos().float().to(device), angle.sin().float().to(device)


def norm_rope(x: torch.Tensor, weight: Optional[torch.Tensor], cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
              positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """rot(x * weight / sqrt(mean(x^2) + eps)) of every row of x [B,H,N,D] (fp16, bf16 or fp32; D 64, 128 or 256), in fp32 and
    rounded once; any strides with contiguous rows, the result is dense.

    weight: [D], or [H,D] for a weight per head, of x's type or fp32; None: no norm.
    cos, sin: fp32 [positions, rotated / 2] (rope_table); None: no rotation.  The first `rotated` elements of a row are turned, a
        multiple of 16 up to D: pairs (i, i + rotated / 2), or (2i, 2i + 1) where interleaved.
    positions: int32 [B,N], or [B] (of every sequence's first token; the others follow), or None (0 to N - 1).  The rotated elements of
        a token whose position is outside the table are NaN, and with them its row's gradient and the weight's: give padding a position
        in the table.
    """
    return _lib.host().norm_rope(x, weight, cos, sin, positions, float(eps), bool(interleaved))


def norm_rope_pair(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], positions: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """norm_rope of queries [B,H,N,D] and keys [B,Hk,N,D] of the same tokens in one launch (and one for their gradients, with a
    small one for the weights')."""
    return _lib.host().norm_rope_pair(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
