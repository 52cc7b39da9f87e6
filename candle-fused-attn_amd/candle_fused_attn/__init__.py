"""candle_fused_attn on MI355X: fused fp32 scaled-dot-product attention, forward and
deterministic backward, head_dim 32, 64 or 128 (the reference's is 64), on hand-written gfx950
kernels (libfattn.so).

The public surface mirrors the reference crate's (src/lib.rs:90-161): `fused_attention`,
`fused_attention_qkv`, `CUDA_HEAD_DIM`. Around them, without a counterpart there: rotary positions
(`fused_rotary`, `fused_rotary_qkv`, `rotary_frequencies`), a paged key-value cache (`paged_append`,
`paged_attention`) and attention to states of another length (`fused_cross_attention`).
"""
from ._lib import FusedAttentionError, LIB_PATH, version
from .cross import fused_cross_attention
from .ops import (
    CUDA_HEAD_DIM,
    HIP_HEAD_DIM,
    HIP_HEAD_DIMS,
    float4_aligned,
    fused_attention,
    fused_attention_qkv,
    qkv_projection_of,
    reads_in_place,
    set_dq_sum,
    set_projection_route,
)
from .paged import paged_append, paged_attention
from .rotary import fused_rotary, fused_rotary_qkv, rotary_frequencies

__all__ = [
    "CUDA_HEAD_DIM",
    "HIP_HEAD_DIM",
    "HIP_HEAD_DIMS",
    "FusedAttentionError",
    "LIB_PATH",
    "float4_aligned",
    "fused_attention",
    "fused_attention_qkv",
    "fused_cross_attention",
    "fused_rotary",
    "fused_rotary_qkv",
    "paged_append",
    "paged_attention",
    "qkv_projection_of",
    "reads_in_place",
    "rotary_frequencies",
    "set_dq_sum",
    "set_projection_route",
    "version",
]
