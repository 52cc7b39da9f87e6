"""A paged key-value cache: the append of new tokens, and the attention of one token over it.

The cache is two tensors the caller owns, k_pages and v_pages, [pages, kv_heads, page_size, d] (any
strides with 16-byte aligned rows; page_size a multiple of 16; d 32, 64 or 128), f32, f16 or bf16. A
page table, [b, width] int32, names each sequence's pages in order: token t of sequence b lies in slot
t % page_size of page table[b, t // page_size]. Lengths are [b] int32 tensors on the device: no call
here copies them to the host or waits. Activations are of the cache's type, or f32.
"""
from __future__ import annotations

import torch

from ._lib import operators


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
    no slot that holds no new token is touched. Two new tokens must not share a slot, and k, v and q must
    not lie in the cache. Not differentiable; a graph that saved the pages before refuses its backward, as
    after any operation in place.
    """
    return operators().paged_append(k, v, k_pages, v_pages, page_table, lengths, counts, q, frequencies,
                                    interleaved, magnitude)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float) -> torch.Tensor:
    """softmax(q k^T scale) v of one token per sequence over its first lengths[b] cached tokens (its
    own among them, once appended).

    q: [b, h, 1, d], of the cache's type or f32, h a multiple of the cache's key heads (query head i
    reads key head i // (h // kv_heads)). Returns [b, h, 1, d] of q's type. A sequence of length 0
    gives 0; one whose length the table cannot hold, or that names a page outside the cache, NaN.
    Infinities and NaN that a token sees give what the formula gives of them. Not differentiable.
    """
    return operators().paged_attention(q, k_pages, v_pages, page_table, lengths, scale)
