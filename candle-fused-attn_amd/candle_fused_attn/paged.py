"""A paged key-value cache: the append of new tokens, and the attention of one token over it.

The cache is two tensors the caller owns, k_pages and v_pages, [pages, kv_heads, page_size, d] (any
strides with 16-byte aligned rows; page_size a multiple of 16; d 32, 64 or 128), f32, f16 or bf16. A
page table, [b, width] int32, names each sequence's pages in order: token t of sequence b lies in slot
t % page_size of page table[b, t // page_size]. Lengths are [b] int32 tensors on the device: no call
here copies them to the host or waits. Activations are of the cache's type, or f32.
"""
from __future__ import annotations

import torch

from . import _lib
from ._call import aligned_rows, launch, pack, require, rows, workspace
from ._lib import FusedAttentionError
from .rotary import check_frequencies

_I32 = (torch.int32,)


def _check_cache(who: str, x, k_pages, v_pages, page_table, lengths, b: int, d: int) -> int:
    """The cache's key heads."""
    require(who, "k_pages", k_pages, 4, x)
    require(who, "v_pages", v_pages, 4, x, (k_pages.dtype,))
    shape = k_pages.shape
    if v_pages.shape != shape or shape[3] != d:
        raise FusedAttentionError(
            f"{who}: k_pages and v_pages [pages, kv_heads, page_size, {d}] expected, got "
            f"{list(k_pages.shape)} and {list(v_pages.shape)}")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.stride(3) != 1 and d > 1:
            raise FusedAttentionError(f"{who}: {name} must have a contiguous last dimension, strides "
                                      f"{list(t.stride())}")
    require(who, "page_table", page_table, 2, x, _I32)
    require(who, "lengths", lengths, 1, x, _I32)
    if page_table.shape[0] != b or lengths.shape[0] != b or not lengths.is_contiguous() or (
            page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise FusedAttentionError(
            f"{who}: a page table [{b}, width] with contiguous rows and contiguous lengths [{b}] "
            f"expected, got {list(page_table.shape)} and {list(lengths.shape)}")
    return shape[1]


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor,
                 counts: torch.Tensor | None = None, q: torch.Tensor | None = None,
                 frequencies: torch.Tensor | None = None, interleaved: bool = False,
                 magnitude: float = 1.0) -> torch.Tensor | None:
    """Writes up to s new tokens per sequence into the cache, in place, in one launch.

    k, v: [b, kv_heads, s, d], any strides. Token i of sequence b (i < counts[b]; counts None: all s)
    becomes its token lengths[b] + i; lengths are what the caches hold before the call, and are not
    changed. With `frequencies` the keys are turned as fused_rotary turns them, at their position
    lengths[b] + i; so is `q` ([b, h, s, d], of k's type), every row of it, and the call returns it (a
    new tensor; None without q). f32 keys and values are rounded to the cache's type. A token whose
    page the table or the cache does not have is not written (its sequence's attention gives NaN), and
    no slot that holds no new token is touched. Two new tokens must not share a slot. Not
    differentiable.
    """
    who = "paged_append"
    require(who, "k", k, 4)
    require(who, "v", v, 4, k, (k.dtype,))
    b, hk, s, d = k.shape
    if v.shape != k.shape:
        raise FusedAttentionError(f"{who}: k and v must share one shape, got {list(k.shape)} and "
                                  f"{list(v.shape)}")
    if _check_cache(who, k, k_pages, v_pages, page_table, lengths, b, d) != hk:
        raise FusedAttentionError(f"{who}: the cache has {k_pages.shape[1]} key heads, k has {hk}")
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (k, v, q, k_pages, v_pages)):
        raise FusedAttentionError(f"{who}: not differentiable (call it under torch.no_grad())")
    heads, out, qp, op, qst, ost = 0, None, 0, 0, (0, 0, 0), (0, 0, 0)
    if q is not None:
        require(who, "q", q, 4, k, (k.dtype,))
        if q.shape[0] != b or q.shape[2:] != k.shape[2:]:
            raise FusedAttentionError(f"{who}: q and k must agree but for their heads, got "
                                      f"{list(q.shape)} and {list(k.shape)}")
        q, heads = rows(q), q.shape[1]
        out = torch.empty_like(q)
        qp, op, qst, ost = q.data_ptr(), out.data_ptr(), q.stride()[:3], out.stride()[:3]
    if counts is not None:
        require(who, "counts", counts, 1, k, _I32)
        if counts.shape[0] != b or not counts.is_contiguous():
            raise FusedAttentionError(f"{who}: contiguous counts [{b}] expected, got "
                                      f"{list(counts.shape)}")
    dim = 0 if frequencies is None else check_frequencies(who, frequencies, d, k)
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if 0 in t.stride()[:3] and any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape)):
            raise FusedAttentionError(f"{who}: {name} is a broadcast view, whose slots share memory")
    k, v = rows(k), rows(v)
    keep, p = pack(*qst, *ost, *k.stride()[:3], *v.stride()[:3], *k_pages.stride()[:3],
                   *v_pages.stride()[:3])
    launch(k, _lib.lib().fattn_paged_append, _lib.DTYPES[k.dtype], _lib.DTYPES[k_pages.dtype], b,
           heads, hk, s, d, qp, p, op, p + 24, k.data_ptr(), p + 48, v.data_ptr(), p + 72,
           k_pages.data_ptr(), p + 96, v_pages.data_ptr(), p + 120, k_pages.shape[0], k_pages.shape[2],
           page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
           counts.data_ptr() if counts is not None else None,
           frequencies.data_ptr() if frequencies is not None else None, dim, bool(interleaved),
           float(magnitude))
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float) -> torch.Tensor:
    """softmax(q k^T scale) v of one token per sequence over its first lengths[b] cached tokens (its
    own among them, once appended).

    q: [b, h, 1, d], of the cache's type or f32, h a multiple of the cache's key heads (query head i
    reads key head i // (h // kv_heads)). Returns [b, h, 1, d] of q's type. A sequence of length 0
    gives 0; one whose length the table cannot hold, or that names a page outside the cache, NaN.
    Infinities and NaN that a token sees give what the formula gives of them. Not differentiable.
    """
    who = "paged_attention"
    require(who, "q", q, 4)
    b, h, s, d = q.shape
    if s != 1:
        raise FusedAttentionError(f"{who}: q [b, h, 1, d] expected, got shape {list(q.shape)}")
    hk = _check_cache(who, q, k_pages, v_pages, page_table, lengths, b, d)
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise FusedAttentionError(f"{who}: not differentiable (call it under torch.no_grad())")
    q = aligned_rows(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    page_size, width = k_pages.shape[2], page_table.shape[1]
    ws, wp, size = workspace(q, "fattn_paged_attention_workspace_bytes", b, h, hk, d, width * page_size)
    keep, p = pack(*q.stride()[:2], *k_pages.stride()[:3], *v_pages.stride()[:3])
    launch(q, _lib.lib().fattn_paged_attention, _lib.DTYPES[q.dtype], _lib.DTYPES[k_pages.dtype], b, h, hk, d,
           q.data_ptr(), p, out.data_ptr(), k_pages.data_ptr(), p + 16, v_pages.data_ptr(), p + 40, k_pages.shape[0], page_size, page_table.data_ptr(),
           page_table.stride(0), width, lengths.data_ptr(), float(scale),
           wp, size)
    return out
