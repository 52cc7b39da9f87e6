"""What the operators around self-attention share in Python: their graphs."""
from __future__ import annotations

import torch

from ._lib import FusedAttentionError


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """A four-dimensional `t` itself where its rows are contiguous and 16-byte aligned, else a contiguous
    copy."""
    per = 16 // t.element_size()
    if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(
            st % per == 0 or n <= 1 for st, n in zip(t.stride()[:3], t.shape)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


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
