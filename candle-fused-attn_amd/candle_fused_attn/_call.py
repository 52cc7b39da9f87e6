"""What the operators around self-attention share: checks of their tensors, and the call itself."""
from __future__ import annotations

import ctypes

import torch

from ._lib import DTYPES, FusedAttentionError, check

A2, A3, A9 = ctypes.c_int64 * 2, ctypes.c_int64 * 3, ctypes.c_int64 * 9
P3 = ctypes.c_void_p * 3


def require(who: str, name: str, t, rank: int, device: torch.device | None = None,
            dtypes=None) -> None:
    """A tensor of `rank` dimensions on a HIP device (that of the first operand), of a type the
    operator takes."""
    if not isinstance(t, torch.Tensor):
        raise FusedAttentionError(f"{who}: {name} must be a tensor")
    if t.dtype not in (DTYPES if dtypes is None else dtypes):
        takes = ", ".join(str(d)[6:] for d in (DTYPES if dtypes is None else dtypes))
        raise FusedAttentionError(f"{who}: {name} must be {takes}, got {str(t.dtype)[6:]}")
    if t.dim() != rank:
        raise FusedAttentionError(f"{who}: {name} must have {rank} dimensions, got shape {list(t.shape)}")
    if t.device.type != "cuda":
        raise FusedAttentionError(f"{who}: {name} is not on a HIP device (this operator has no CPU path)")
    if device is not None and t.device != device:
        raise FusedAttentionError(f"{who}: {name} is on {t.device}, the first operand on {device}")


def rows(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where head_dim is contiguous, else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where its rows are contiguous and 16-byte aligned, else a contiguous copy."""
    per = 16 // t.element_size()
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and all(
            s % per == 0 for s, n in zip(st[:-1], t.shape) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def strides3(t: torch.Tensor):
    return A3(*t.stride()[:3])


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
