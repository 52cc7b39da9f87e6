"""Rotary positions: heads turned, pair by pair, by an angle of their position, before attention.

A head's first `dim` values are dim / 2 pairs, (i, i + dim / 2) or, interleaved, (2 i, 2 i + 1); pair i
at position p turns by p * frequencies[i] radians and is scaled by `magnitude`; values past dim stay.
Angles are formed and reduced in 64 bits, so far positions keep their precision, and there is no
largest position. f32, f16 and bf16; computed in 32 bits and rounded once.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._call import launch, pack, require, rows
from ._lib import FusedAttentionError

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


_F64 = (torch.float64,)
_INTS = (torch.int64, torch.int32)


def check_frequencies(who: str, frequencies, d: int, like: torch.Tensor) -> int:
    """The rotated part of a head of d values."""
    require(who, "frequencies", frequencies, 1, like, _F64)
    dim = 2 * frequencies.shape[0]
    if dim > d or not frequencies.is_contiguous():
        raise FusedAttentionError(f"{who}: contiguous frequencies of at most {d // 2} pairs expected, "
                                  f"got {frequencies.shape[0]}")
    return dim


def _forward(xs, heads, positions, frequencies, interleaved, magnitude, inverse):
    """heads 0: xs are one or two [b, h, s, d] operands, all turned; else the one [b, s, 3 h d]
    projection, whose q and k are turned and v copied. New tensors."""
    ys = [torch.empty_like(x) for x in xs]
    x, y = xs[0], ys[0]
    xp, yp = x.data_ptr(), y.data_ptr()
    if heads:
        b, s, w = x.shape
        d = w // (3 * heads)
        step = heads * d * x.element_size()
        (xb, xs_, _), (yb, ys_, _) = x.stride(), y.stride()
        sizes = (heads, heads, heads)
        at = (xp, xp + step, xp + 2 * step, yp, yp + step, yp + 2 * step)
        strides = (xb, d, xs_) * 3 + (yb, d, ys_) * 3
        rotated = 0b011
    else:
        b, h, s, d = x.shape
        rotated = 0b111
        if len(xs) == 2:
            x2, y2 = xs[1], ys[1]
            sizes = (h, x2.shape[1], 0)
            at = (xp, x2.data_ptr(), 0, yp, y2.data_ptr(), 0)
            strides = (*x.stride()[:3], *x2.stride()[:3], 0, 0, 0, *y.stride()[:3], *y2.stride()[:3],
                       0, 0, 0)
        else:
            sizes, at = (h, 0, 0), (xp, 0, 0, yp, 0, 0)
            strides = (*x.stride()[:3], *(0,) * 6, *y.stride()[:3], *(0,) * 6)
    if positions.dim() == 1:
        pb, ps = 0, positions.stride(0)
    else:
        pb, ps = positions.stride()
        if positions.shape[0] == 1:
            pb = 0
    keep, p = pack(*sizes, *at, *strides, pb, ps)
    launch(x, _lib.lib().fattn_rotary, _lib.DTYPES[x.dtype], b, s, d, p, p + 24, p + 48, p + 72, p + 144,
           rotated, positions.data_ptr(), 64 if positions.dtype == torch.int64 else 32, p + 216,
           frequencies.data_ptr(), 2 * frequencies.shape[0], interleaved, magnitude, inverse)
    return ys


class _Rotary(torch.autograd.Function):
    """The turn; its gradient is the turn back, by the same Function where a graph of it is asked for (so
    it can be differentiated again)."""

    @staticmethod
    def forward(ctx, positions, frequencies, heads, interleaved, magnitude, inverse, *xs):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (heads, interleaved, magnitude, inverse)
        ctx.set_materialize_grads(False)
        ys = _forward(xs, heads, positions, frequencies, interleaved, magnitude, inverse)
        return ys[0] if len(ys) == 1 else tuple(ys)

    @staticmethod
    def backward(ctx, *grads):
        positions, frequencies = ctx.saved_tensors
        heads, interleaved, magnitude, inverse = ctx.how
        need = ctx.needs_input_grad
        # (A projection's gradient is read by its heads: any strides but for the last dimension.)
        at = [i for i, g in enumerate(grads) if g is not None and need[6 + i]]
        out = [None] * (6 + len(grads))
        if at:
            turned = _apply([rows(grads[i]) for i in at], heads, positions, frequencies, interleaved,
                            magnitude, not inverse)
            for i, g in zip(at, turned):
                out[6 + i] = g
        return tuple(out)


def _apply(xs, heads, positions, frequencies, interleaved, magnitude, inverse):
    if torch.is_grad_enabled() and (xs[0].requires_grad or xs[-1].requires_grad):
        ys = _Rotary.apply(positions, frequencies, heads, interleaved, magnitude, inverse, *xs)
        return (ys,) if len(xs) == 1 else ys
    return _forward(xs, heads, positions, frequencies, interleaved, magnitude, inverse)


def _check_positions(who: str, positions, b: int, s: int, like: torch.Tensor) -> None:
    if not isinstance(positions, torch.Tensor) or positions.dim() not in (1, 2):
        raise FusedAttentionError(f"{who}: positions must be a [s] or [b, s] tensor")
    require(who, "positions", positions, positions.dim(), like, _INTS)
    if positions.shape[-1] != s or (positions.dim() == 2 and positions.shape[0] not in (1, b)):
        raise FusedAttentionError(f"{who}: positions [{s}] or [{b}, {s}] expected, got shape "
                                  f"{list(positions.shape)}")


def fused_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                 frequencies: torch.Tensor, interleaved: bool = False,
                 magnitude: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k with their positions turned into them, in one launch; differentiable in q and k.

    q: [b, h, s, d], k: [b, kv_heads, s, d], of one type (f32, f16 or bf16), any strides (copied first
    where head_dim is not contiguous); positions: [s] or [b, s], int64 or int32; frequencies: float64,
    one per pair of the rotated part of a head (rotary_frequencies). The results have the operands'
    shapes and types.
    """
    who = "fused_rotary"
    require(who, "q", q, 4)
    require(who, "k", k, 4, q, (q.dtype,))
    b, _, s, d = q.shape
    if k.shape[0] != b or k.shape[2:] != q.shape[2:]:
        raise FusedAttentionError(f"{who}: q and k must agree but for their heads, got {list(q.shape)} "
                                  f"and {list(k.shape)}")
    _check_positions(who, positions, b, s, q)
    check_frequencies(who, frequencies, d, q)
    q2, k2 = _apply([rows(q), rows(k)], 0, positions, frequencies, bool(interleaved),
                    float(magnitude), False)
    return q2, k2


def fused_rotary_qkv(qkv: torch.Tensor, heads: int, positions: torch.Tensor,
                     frequencies: torch.Tensor, interleaved: bool = False,
                     magnitude: float = 1.0) -> torch.Tensor:
    """fused_rotary on the q and k of a fused [b, s, 3 h d] projection laid out [q | k | v]: a new
    projection, v copied, which fused_attention_qkv takes; differentiable, with one gradient shaped
    like qkv."""
    who = "fused_rotary_qkv"
    require(who, "qkv", qkv, 3)
    b, s, w = qkv.shape
    heads = int(heads)
    if heads <= 0 or w == 0 or w % (3 * heads) != 0:
        raise FusedAttentionError(f"{who}: last dimension {w} is not 3 x {heads} heads x head_dim")
    _check_positions(who, positions, b, s, qkv)
    check_frequencies(who, frequencies, w // 3 // heads, qkv)
    return _apply([rows(qkv)], heads, positions, frequencies, bool(interleaved), float(magnitude),
                  False)[0]
