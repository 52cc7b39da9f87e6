"""Self-attention whose scores are capped, lowered by distance, or masked by documents and prefixes, fp32.

As fused_attention, with shared key heads, and queries that may be the last of a longer context: a prompt's
next chunk over what came before it.
"""
from __future__ import annotations

import torch

from ._lib import operators


def fused_scored_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool,
                           cap: float | None = None, slopes: torch.Tensor | None = None,
                           documents: torch.Tensor | None = None,
                           prefix: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(y) v over the keys that a query sees, y the score x = scale q.k, with `cap` (1e-30 to 1e30)
    taken as cap tanh(x / cap), and with `slopes` ([h] f32, finite, one per query head) lowered by the slope times the
    distance |i - j| of the positions (a negative slope times the largest distance has to be finite too).

    q: [b, h, sq, d], the last sq of sk positions, k, v: [b, kv_heads, sk, d] f32 on one HIP device, any
    strides (copied first when the kernels cannot read them in place), d 32, 64 or 128, h a multiple of
    kv_heads (query head i reads key head i // (h // kv_heads)). When `causal` a query sees the keys at its
    position and before it, and with `prefix` ([b] int32; one outside [0, sk] counts as the nearest) the
    sample's first prefix[b] too; else all. With `documents` ([b, sk] int32 ids with contiguous rows) a token
    sees and is seen by tokens of its own id only, and one of a negative id (padding) by and of none; ids in
    order, as of documents packed one after the other, leave each its own keys to walk. Returns [b, h, sq, d],
    laid out as a contiguous [b, sq, h, d] buffer; a query that sees no key gives 0. Differentiable in q, k
    and v, once, in reverse mode (a forward-mode tangent is refused, and slopes that require a gradient
    where a graph is recorded).
    """
    return operators().scored_attention(q, k, v, scale, causal, cap, slopes, documents, prefix)
