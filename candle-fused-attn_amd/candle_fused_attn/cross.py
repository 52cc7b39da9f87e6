"""Cross attention: a decoder's queries to an encoder's states of another length, fp32.

As fused_attention, with keys and values of their own length and number of heads, and per-sample key
lengths in place of a mask.
"""
from __future__ import annotations

import torch

from . import _lib
from ._call import aligned_rows, launch, not_twice, pack, require, workspace
from ._lib import FusedAttentionError

_F32 = (torch.float32,)
_I32 = (torch.int32,)


def _forward(q, k, v, scale, key_lengths):
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    L = _lib.lib()
    out, lse = q.new_empty((b, sq, h, d)), q.new_empty((b, h, sq))
    ws, wp, size = workspace(q, "fattn_cross_workspace_bytes", b, h, hk, sq, sk, d)
    keep, p = pack(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    launch(q, L.fattn_cross_forward, q.data_ptr(), p, k.data_ptr(), p + 24, v.data_ptr(), p + 48, b, h, hk, sq, sk, d,
           key_lengths.data_ptr() if key_lengths is not None else None, scale, out.data_ptr(),
           lse.data_ptr(), wp, size)
    return out, lse


class _FusedCrossAttention(torch.autograd.Function):
    """[b, h, sq, d] and [b, kv_heads, sk, d] in, the [b, h, sq, d] view of the output out."""

    @staticmethod
    def forward(ctx, q, k, v, scale, key_lengths):
        out, lse = _forward(q, k, v, scale, key_lengths)
        ctx.save_for_backward(q, k, v, key_lengths, out, lse)
        ctx.scale = scale
        return out.transpose(1, 2)

    @staticmethod
    def backward(ctx, grad):
        q, k, v, key_lengths, out, lse = ctx.saved_tensors
        with_graph = torch.is_grad_enabled()
        if with_graph:
            inputs, grad = (q, k, v, grad), grad.detach()
        grad = aligned_rows(grad)
        b, h, sq, d = q.shape
        hk, sk = k.shape[1], k.shape[2]
        dq, dkv = q.new_empty((b, sq, h, d)), q.new_empty((b, sk, 2, hk, d))
        keep, p = pack(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *grad.stride()[:3])
        ws, wp, size = workspace(q, "fattn_cross_backward_workspace_bytes", b, h, hk, sq, sk, d)
        launch(q, _lib.lib().fattn_cross_backward, q.data_ptr(), p, k.data_ptr(), p + 24, v.data_ptr(),
               p + 48, b, h, hk, sq, sk, d,
               key_lengths.data_ptr() if key_lengths is not None else None, ctx.scale, out.data_ptr(),
               lse.data_ptr(), grad.data_ptr(), p + 72, dq.data_ptr(), dkv.data_ptr(), wp, size)
        dk, dv = dkv.transpose(1, 3).unbind(2)  # [b, kv_heads, sk, d] each
        grads = dq.transpose(1, 2), dk, dv
        if with_graph:
            grads = not_twice("fused_cross_attention", inputs, grads)
        return *grads, None, None


def fused_cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                          key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v, each sample seeing its first key_lengths[b] keys (None: all).

    q: [b, h, sq, d], k, v: [b, kv_heads, sk, d] f32 on one HIP device, any strides (copied first when
    the kernels cannot read them in place), d 32, 64 or 128, h a multiple of kv_heads (query head i
    reads key head i // (h // kv_heads)); key_lengths: [b] int32 (one outside [0, sk] counts as the
    nearest). Returns [b, h, sq, d], a transposed view of a contiguous [b, sq, h, d] buffer; a sample
    that sees no key gives 0.
    """
    who = "fused_cross_attention"
    require(who, "q", q, 4, None, _F32)
    require(who, "k", k, 4, q, _F32)
    require(who, "v", v, 4, q, _F32)
    b, h, _, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise FusedAttentionError(f"{who}: q [b, h, sq, d] and k, v [b, kv_heads, sk, d] expected, got "
                                  f"{list(q.shape)} {list(k.shape)} {list(v.shape)}")
    if key_lengths is not None:
        require(who, "key_lengths", key_lengths, 1, q, _I32)
        if key_lengths.shape[0] != b or not key_lengths.is_contiguous():
            raise FusedAttentionError(f"{who}: contiguous key_lengths [{b}] expected, got "
                                      f"{list(key_lengths.shape)}")
    q, k, v = aligned_rows(q), aligned_rows(k), aligned_rows(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _FusedCrossAttention.apply(q, k, v, float(scale), key_lengths)
    return _forward(q, k, v, float(scale), key_lengths)[0].transpose(1, 2)
