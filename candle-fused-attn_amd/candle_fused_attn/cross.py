"""Cross attention: a decoder's queries to an encoder's states of another length, fp32.

As fused_attention, with keys and values of their own length and number of heads, and per-sample key
lengths in place of a mask.
"""
from __future__ import annotations

import torch

from ._lib import operators


def fused_cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                          key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v, each sample seeing its first key_lengths[b] keys (None: all).

    q: [b, h, sq, d], k, v: [b, kv_heads, sk, d] f32 on one HIP device, any strides (copied first when
    the kernels cannot read them in place), d 32, 64 or 128, h a multiple of kv_heads (query head i
    reads key head i // (h // kv_heads)); key_lengths: [b] int32 (one outside [0, sk] counts as the
    nearest). Returns [b, h, sq, d], laid out as a contiguous [b, sq, h, d] buffer; a sample that sees no
    key gives 0. Differentiable once, in reverse mode (a forward-mode tangent is refused).
    """
    return operators().cross_attention(q, k, v, scale, key_lengths)
