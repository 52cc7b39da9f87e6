"""Cross attention on the GPU against its formula in 64 bits: lengths of queries and keys around the
kernels' tiles, grouped heads, per-sample key lengths (0 among them), strides, garbage behind the last
key, scale signs.

Tolerance: the bar of the fp32 attentions here, 2e-6 normwise on N(0, 1) inputs, for every output."""
from __future__ import annotations

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu

TOL = 2e-6


def rel(x, ref):
    n = float(ref.double().cpu().norm())
    return float((x.double().cpu() - ref.double().cpu()).norm()) / n if n else float(x.abs().max())


def operands(dev, b, h, hk, sq, sk, d, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, g = (torch.randn(b, sq, h, d, generator=gen).to(dev).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(b, sk, hk, d, generator=gen).to(dev).transpose(1, 2) for _ in range(2))
    return q, k, v, g


def formula(q, k, v, scale, lengths=None):
    """The output in 64 bits on the CPU, differentiable."""
    h, hk, sk = q.shape[1], k.shape[1], k.shape[2]
    k, v = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    x = torch.matmul(q, k.transpose(2, 3)) * scale
    if lengths is None:
        return torch.matmul(torch.softmax(x, -1), v)
    gone = torch.arange(sk)[None, None, None, :] >= torch.tensor(lengths)[:, None, None, None]
    p = torch.softmax(x.masked_fill(gone, -1e300), -1).masked_fill(gone, 0.0)
    return torch.matmul(p, v.masked_fill(gone.transpose(2, 3), 0.0))


def ints(dev, lengths):
    return None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)


SHAPES = [  # b, h, hk, sq, sk, d, lengths
    (1, 1, 1, 1, 1, 64, None), (2, 3, 3, 1, 1000, 64, None), (8, 6, 6, 1, 1537, 64, None),
    (2, 4, 2, 3, 33, 32, [33, 7]), (3, 4, 1, 5, 700, 128, [0, 1, 700]), (1, 8, 8, 31, 64, 64, None),
    (2, 2, 2, 33, 31, 64, None), (2, 6, 3, 240, 333, 64, [333, 100]), (1, 4, 4, 128, 129, 128, None),
    (2, 8, 2, 257, 512, 32, [511, 0]), (4, 2, 1, 17, 65, 64, [65, 64, 33, 32]),
    (300, 1, 1, 20, 40, 64, None), (300, 1, 1, 64, 50, 32, None), (70, 4, 2, 70, 20, 128, None),
]


@pytest.mark.parametrize("b,h,hk,sq,sk,d,lengths", SHAPES)
def test_forward(cuda, b, h, hk, sq, sk, d, lengths):
    q, k, v, _ = operands(cuda, b, h, hk, sq, sk, d)
    for scale in (d ** -0.5, -1.0 / 16):
        out = cfa.fused_cross_attention(q, k, v, scale, ints(cuda, lengths))
        assert out.shape == q.shape and out.transpose(1, 2).is_contiguous()
        ref = formula(*(t.double().cpu() for t in (q, k, v)), scale, lengths)
        assert rel(out, ref) <= TOL
        for i, n in enumerate(lengths or []):
            if n == 0:
                assert float(out[i].abs().max()) == 0.0
        assert torch.equal(out, cfa.fused_cross_attention(q, k, v, scale, ints(cuda, lengths)))
