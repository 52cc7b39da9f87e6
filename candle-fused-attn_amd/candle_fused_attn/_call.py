"""What the operators around self-attention share: checks of their tensors, and the call itself."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import DTYPES, FusedAttentionError, check

ALL = tuple(DTYPES)
_ARRAYS = {n: ctypes.c_int64 * n for n in range(1, 40)}


def pack(*values):
    """One int64 array of `values` (sizes, strides, addresses) and its address, which the C entries take
    parts of: on small calls the host is the whole time, and an array per operand costs it 0.4 us each.
    (Keep the array until the call returns.)"""
    a = _ARRAYS[len(values)](*values)
    return a, ctypes.addressof(a)


def require(who: str, name: str, t, rank: int, like: torch.Tensor | None = None, dtypes=ALL) -> None:
    """A tensor of `rank` dimensions on a HIP device (that of `like`), of a type the operator takes."""
    if (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == rank and t.is_cuda
            and (like is None or t.get_device() == like.get_device())):
        return
    if not isinstance(t, torch.Tensor):
        raise FusedAttentionError(f"{who}: {name} must be a tensor")
    if t.dtype not in dtypes:
        takes = ", ".join(str(d)[6:] for d in dtypes)
        raise FusedAttentionError(f"{who}: {name} must be {takes}, got {str(t.dtype)[6:]}")
    if t.dim() != rank:
        raise FusedAttentionError(f"{who}: {name} must have {rank} dimensions, got shape {list(t.shape)}")
    if not t.is_cuda:
        raise FusedAttentionError(f"{who}: {name} is not on a HIP device (this operator has no CPU path)")
    raise FusedAttentionError(f"{who}: {name} is on {t.device}, the first operand on {like.device}")


def rows(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where head_dim is contiguous, else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """A four-dimensional `t` itself where its rows are contiguous and 16-byte aligned, else a contiguous
    copy."""
    per = 15 // t.element_size()
    s0, s1, s2, s3 = t.stride()
    if s3 == 1 and not (s0 | s1 | s2) & per and not t.data_ptr() & 15:
        return t
    if s3 == 1 and not t.data_ptr() & 15 and not any(
            s & per for s, n in zip((s0, s1, s2), t.shape) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def launch(t: torch.Tensor, fn, *args) -> None:
    """fn(*args, stream) on torch's current stream of t's device, with that device current."""
    index = t.get_device()
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(query: str, *sizes: int) -> int:
    """A C size query (a function of the sizes alone)."""
    return getattr(_lib.lib(), query)(*sizes)


def workspace(t: torch.Tensor, query: str, *sizes: int):
    """The workspace of a call, from torch's allocator: (tensor, address, bytes), or (None, None, 0)."""
    size = _workspace_bytes(query, *sizes)
    if not size:
        return None, None, 0
    ws = torch.empty(size, dtype=torch.uint8, device=t.device)
    return ws, ws.data_ptr(), size


class _NotTwice(torch.autograd.Function):
    """Gradients that were asked for with a graph: they are not differentiable, and say so when it is
    tried (without this they would look like constants)."""

    @staticmethod
    def forward(ctx, who, n, *tensors):
        ctx.who = who
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise FusedAttentionError(f"{ctx.who}: its gradient is not differentiable")


def not_twice(who: str, inputs, grads):
    """`grads` as results of a node on `inputs` that refuses to be differentiated."""
    return _NotTwice.apply(who, len(grads), *grads, *inputs)
