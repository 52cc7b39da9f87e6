"""A paged key-value cache: the append of new tokens, the attention of one token over it, and tokens back
out of it.

The cache is two tensors the caller owns, k_pages and v_pages, [pages, kv_heads, page_size, d] (any
strides with 16-byte aligned rows; page_size a multiple of 16; d 32, 64 or 128), f32, f16 or bf16; or, in 4
bits, [pages, kv_heads, page_size, fp4_row_bytes(d)] uint8 (rows 4-byte aligned). A
page table, [b, width] int32, names each sequence's pages in order: token t of sequence b lies in slot
t % page_size of page table[b, t // page_size]. Lengths are [b] int32 tensors on the device: no call
here copies them to the host or waits. Activations are of the cache's type, or f32; of any type over a 4-bit
cache.

A 4-bit cache holds a sign and a magnitude of 0, .5, 1, 1.5, 2, 3, 4 or 6 per value, times a power of two per
32 values of a row: the least under which none of them passes 7. An append takes the nearest (the even code
of two), so a value is off by half a step at most: a quarter of the power of two near 0, one of it at 6. A
group of 32 that has a value that is not finite becomes NaN. Values of 3.5 x 2^126 (2.98e38) and more, with which
a group has the power 2^126, become 4 x 2^126, which no float holds: an infinity where the cache is read or attended
over; keys turned past the largest float count as that. d 128 takes 68 bytes, of 256 in 16 bits.
"""
from __future__ import annotations

import torch

from ._lib import DTYPES, FusedAttentionError, operators


def fp4_row_bytes(head_dim: int) -> int:
    """The last dimension of a 4-bit cache's pages: bytes per token and key head."""
    if head_dim not in (32, 64, 128):
        raise FusedAttentionError(f"fp4_row_bytes: the HIP kernels take head_dim 32, 64 or 128, got {head_dim}")
    return head_dim // 2 + 4


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
    new tensor; None without q). f32 keys and values are rounded to the cache's type; a 4-bit cache's codes
    are the nearest to the keys as turned in 64 bits. A token whose
    page the table or the cache does not have is not written (its sequence's attention gives NaN), and
    no slot that holds no new token is touched. Two new tokens must not share a slot, and k, v and q must
    not lie in the cache. Not differentiable; a graph that saved the pages before refuses its backward, as
    after any operation in place.
    """
    return operators().paged_append(k, v, k_pages, v_pages, page_table, lengths, counts, q, frequencies,
                                    interleaved, magnitude)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                    cap: float | None = None, slopes: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v of one token per sequence over its first lengths[b] cached tokens (its
    own among them, once appended). With `cap` a score x is taken as cap tanh(x / cap); with `slopes`
    ([h] f32, one per query head) it is lowered by the slope times the distance lengths[b] - 1 - j to
    token j: what fused_scored_attention does of a sequence's last token.

    q: [b, h, 1, d], of the cache's type or f32 (any over a 4-bit cache), h a multiple of the cache's key
    heads (query head i reads key head i // (h // kv_heads)). Returns [b, h, 1, d] of q's type. A sequence of
    length 0 gives 0; one whose length the table cannot hold, or that names a page outside the cache, NaN.
    Infinities and NaN that a token sees give what the formula gives of them. Not differentiable.
    """
    return operators().paged_attention(q, k_pages, v_pages, page_table, lengths, scale, cap, slopes)


def paged_read(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
               lengths: torch.Tensor, s: int, starts: torch.Tensor | None = None,
               dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens starts[b] + i, i < s (starts, [b] int32; None: from token 0), of each sequence out of the
    cache: k and v, new contiguous [b, kv_heads, s, d] tensors, for the attention of a prompt's next chunk
    over what came before it.

    dtype: f32, f16 or bf16 (None: the cache's type, bf16 of a 4-bit one, which holds its values exactly);
    values that it does not hold are rounded once. Tokens from lengths[b] on, and before token 0, are 0; a
    token that the sequence holds but the table or the cache has no page for is NaN. Not differentiable.
    """
    if dtype is not None and dtype not in DTYPES:
        raise FusedAttentionError(f"paged_read: dtype must be float32, float16 or bfloat16, got {dtype}")
    return operators().paged_read(k_pages, v_pages, page_table, lengths, s, starts,
                                  -1 if dtype is None else DTYPES[dtype])
