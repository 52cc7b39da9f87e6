"""Rotary positions: heads turned, pair by pair, by an angle of their position, before attention.

A head's first `dim` values are dim / 2 pairs, (i, i + dim / 2) or, interleaved, (2 i, 2 i + 1); pair i
at position p turns by p * frequencies[i] radians and is scaled by `magnitude`; values past dim stay.
Angles are formed and reduced in 64 bits, so far positions keep their precision, and there is no
largest position. f32, f16 and bf16; computed in 32 bits and rounded once.
"""
from __future__ import annotations

import math

import torch

from ._lib import FusedAttentionError, operators

_SCALINGS = (None, "linear", "base", "ramp")


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str | None = None,
                       factor: float = 1.0, original_length: int = 4096, low: float = 1.0,
                       high: float = 32.0, device=None) -> torch.Tensor:
    """The dim / 2 frequencies base^(-2 i / dim), radians per position, float64. For contexts `factor`
    times longer than the `original_length` a model was trained on:
      "linear": every frequency divided by the factor;
      "base":   base * factor^(dim / (dim - 2)): the slowest pair is slowed by the factor, the fastest
                stays;
      "ramp":   pairs of at most `low` turns over original_length are divided by the factor, those of
                at least `high` stay, a straight line between.
    """
    who = "rotary_frequencies"
    if dim <= 0 or dim % 2 != 0 or not base > 0.0 or not factor > 0.0:
        raise FusedAttentionError(f"{who}: an even dim and a positive base and factor expected, got "
                                  f"{dim}, {base}, {factor}")
    if scaling not in _SCALINGS:
        raise FusedAttentionError(f"{who}: scaling must be one of {_SCALINGS}, got {scaling!r}")
    if scaling == "ramp" and not (original_length > 0 and high > low):
        raise FusedAttentionError(f"{who}: a positive original_length and low < high expected")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    f = torch.exp(i * (-math.log(base) / dim))
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        keep = ((original_length / (2 * math.pi) * f - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f.to(device) if device is not None else f


def fused_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                 frequencies: torch.Tensor, interleaved: bool = False,
                 magnitude: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k with their positions turned into them, in one launch; differentiable in q and k (in reverse
    mode: a forward-mode tangent is refused).

    q: [b, h, s, d], k: [b, kv_heads, s, d], of one type (f32, f16 or bf16), any strides (copied first
    where head_dim is not contiguous); positions: [s] or [b, s], int64 or int32; frequencies: float64,
    one per pair of the rotated part of a head (rotary_frequencies), constants: ones that require a
    gradient are refused where a graph is recorded. The results have the operands' shapes and types.
    """
    return operators().rotary(q, k, positions, frequencies, interleaved, magnitude)


def fused_rotary_qkv(qkv: torch.Tensor, heads: int, positions: torch.Tensor,
                     frequencies: torch.Tensor, interleaved: bool = False,
                     magnitude: float = 1.0) -> torch.Tensor:
    """fused_rotary on the q and k of a fused [b, s, 3 h d] projection laid out [q | k | v]: a new
    projection, v copied, which fused_attention_qkv takes; differentiable, with one gradient shaped
    like qkv."""
    return operators().rotary_qkv(qkv, int(heads), positions, frequencies, interleaved, magnitude)
