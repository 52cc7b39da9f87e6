"""Rotary positions on the GPU against the formula in 64 bits: layouts, partial heads, types, far
positions, strides, gradients (against the formula's, and against differences), graphs.

Tolerance: y = x0 c - x1 s takes four roundings of 2^-24 (c, s, a product, the sum), each of at most
(|x0| + |x1|) magnitude, and half a step of a 16-bit result."""
from __future__ import annotations

import math

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def formula(x, positions, f, interleaved, magnitude=1.0, sign=1.0):
    """x [b, h, s, d] turned, 64 bits on the CPU."""
    x, f = x.double().cpu(), f.cpu()
    pos = positions.cpu().double()
    a = (pos if pos.dim() == 2 else pos[None])[:, None, :, None] * f
    n = f.numel()
    i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    c, s, y = magnitude * a.cos(), sign * magnitude * a.sin(), x.clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def near(got, ref, x, magnitude=1.0):
    eps = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    size = 2 * max(1.0, magnitude) * x.double().cpu().abs().amax(-1, keepdim=True)
    err = (got.double().cpu() - ref).abs()
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0  # half a step of subnormal f16
    assert bool((err <= 4 * 2.0 ** -24 * size + eps * 1.0001 * ref.abs() + tiny).all()), float(err.max())


def operands(dev, dtype, b, h, hk, s, d, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(b, s, n, d, generator=gen).to(dtype).to(dev).transpose(1, 2) for n in (h, hk)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d,dim", [(64, 64), (128, 64), (32, 8), (80, 20), (96, 2), (64, 0), (10, 6)])
def test_forward(cuda, dtype, d, dim, interleaved):
    b, h, hk, s = 2, 5, 2, 37
    q, k = operands(cuda, dtype, b, h, hk, s, d)
    f = cfa.rotary_frequencies(dim, device=cuda) if dim else torch.empty(0, dtype=torch.float64,
                                                                         device=cuda)
    pos = torch.randint(0, 5000, (b, s), device=cuda)
    for magnitude in (1.0, 1.3):
        got = cfa.fused_rotary(q, k, pos, f, interleaved, magnitude)
        for x, y in zip((q, k), got):
            assert y.dtype == dtype and y.shape == x.shape
            near(y, formula(x, pos, f, interleaved, magnitude), x, magnitude)


@pytest.mark.parametrize("b,h,hk,s", [(1, 1, 1, 1), (1, 32, 8, 1), (64, 6, 6, 1), (3, 1, 1, 1000),
                                      (1, 70, 3, 129), (40, 2, 2, 100)])
def test_sizes(cuda, b, h, hk, s):
    q, k = operands(cuda, torch.float32, b, h, hk, s, 64, seed=1)
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.arange(s, device=cuda, dtype=torch.int32)
    for x, y in zip((q, k), cfa.fused_rotary(q, k, pos, f)):
        near(y, formula(x, pos, f, False), x)


def test_far_positions(cuda):
    """Angles to 1e9 radians, either sign: the 64-bit product's half step, 2^-53 of the angle, is 1e-7."""
    q, k = operands(cuda, torch.float32, 1, 2, 1, 6, 64, seed=2)
    f = cfa.rotary_frequencies(64, device=cuda)
    pos = torch.tensor([[0, 131071, -131071, 2 ** 24 + 1, 10 ** 7, -(10 ** 9)]], device=cuda)
    for x, y in zip((q, k), cfa.fused_rotary(q, k, pos, f)):
        err = (y.double().cpu() - formula(x, pos, f, False)).abs()
        assert float(err.max()) <= 5 * (4 * 2.0 ** -24 * 2 + 3 * 1.2e-7 * 2)


def test_layouts(cuda):
    """Contiguous heads, padded rows, broadcast operands, odd offsets, a head_dim that is not contiguous:
    the same values bit for bit."""
    b, h, s, d = 2, 3, 20, 64
    q, k = operands(cuda, torch.float32, b, h, h, s, d, seed=3)
    f, pos = cfa.rotary_frequencies(32, device=cuda), torch.arange(s, device=cuda)
    want = cfa.fused_rotary(q, k, pos, f)
    padded = torch.zeros(b, h, s, d + 5, device=cuda)
    padded[..., 1:d + 1] = q
    for x in (q.contiguous(), padded[..., 1:d + 1], q.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)):
        got = cfa.fused_rotary(x, k, pos, f)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = cfa.fused_rotary(q, k[:, :1].expand(b, h, s, d), pos[None].expand(b, s), f)
    assert torch.equal(got[1], want[1][:, :1].expand(b, h, s, d))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients(cuda, dtype, interleaved):
    """Each operand's gradient is its output's, turned back; an operand that needs none has none, an
    output without a gradient gives none."""
    q, k = operands(cuda, dtype, 2, 4, 2, 33, 64, seed=4)
    gq, gk = operands(cuda, dtype, 2, 4, 2, 33, 64, seed=5)
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.arange(100, 133, device=cuda)
    q.requires_grad_(), k.requires_grad_()
    yq, yk = cfa.fused_rotary(q, k, pos, f, interleaved, 1.1)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    near(dq, formula(gq, pos, f, interleaved, 1.1, -1.0), gq, 1.1)
    near(dk, formula(gk, pos, f, interleaved, 1.1, -1.0), gk, 1.1)
    yq, yk = cfa.fused_rotary(q, k.detach(), pos, f, interleaved, 1.1)
    assert not torch.equal(yk, k) and torch.equal(torch.autograd.grad(yq, q, gq)[0], dq)
    yq, yk = cfa.fused_rotary(q, k, pos, f, interleaved, 1.1)
    assert torch.equal(torch.autograd.grad(yk, k, gk)[0], dk)
    yq, yk = cfa.fused_rotary(q, k, pos, f, interleaved, 1.1)
    assert torch.equal(torch.autograd.grad(yq, q, gq[:, :1].expand_as(gq))[0][:, 0], dq[:, 0])


def test_gradient_against_differences(cuda):
    """The loss is linear in q: its change under a step is the gradient's product with the step."""
    q, k = operands(cuda, torch.float32, 1, 2, 2, 9, 32, seed=6)
    g, step = operands(cuda, torch.float32, 1, 2, 2, 9, 32, seed=7)
    f, pos = cfa.rotary_frequencies(32, device=cuda), torch.arange(9, device=cuda)
    q.requires_grad_()
    out = cfa.fused_rotary(q, k, pos, f)[0]
    (dq,) = torch.autograd.grad(out, q, g, create_graph=True)
    more = cfa.fused_rotary(q.detach() + step, k, pos, f)[0]
    change = float(((more - out).double() * g).sum())
    # 1152 values of about 1, each off by 8 x 2^-24 or less.
    assert abs(change - float((dq.double() * step).sum())) <= 1152 * 8 * 2.0 ** -24
    assert dq.requires_grad is False or dq.grad_fn is not None


def test_gradient_of_the_gradient(cuda):
    """The gradient is linear in the output's gradient, and differentiable in it."""
    q, k = operands(cuda, torch.float32, 1, 2, 2, 5, 32, seed=8)
    g, u = operands(cuda, torch.float32, 1, 2, 2, 5, 32, seed=9)
    f, pos = cfa.rotary_frequencies(32, device=cuda), torch.arange(5, device=cuda)
    q.requires_grad_(), g.requires_grad_()
    out = cfa.fused_rotary(q, k, pos, f)[0]
    (dq,) = torch.autograd.grad(out, q, g, create_graph=True)
    (dg,) = torch.autograd.grad(dq, g, u)
    assert torch.equal(dg, cfa.fused_rotary(u, k, pos, f)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_projection(cuda, dtype):
    """fused_rotary_qkv: q and k of the projection as fused_rotary turns them, v as it is, one gradient;
    a projection whose last dimension is not contiguous is copied."""
    b, s, h, d = 3, 50, 4, 64
    x = torch.randn(b, s, 3 * h * d, device=cuda).to(dtype)
    f, pos = cfa.rotary_frequencies(d, device=cuda), torch.randint(0, 999, (b, s), device=cuda)
    q, k, v = (t.transpose(1, 2) for t in x.view(b, s, 3, h, d).unbind(2))
    want = torch.stack([t.transpose(1, 2) for t in (*cfa.fused_rotary(q, k, pos, f), v)], 2).view(b, s, -1)
    x.requires_grad_()
    out = cfa.fused_rotary_qkv(x, h, pos, f)
    assert torch.equal(out, want)
    g = torch.randn_like(x)
    (dx,) = torch.autograd.grad(out, x, g)
    dq, dk, dv = (t.transpose(1, 2) for t in dx.view(b, s, 3, h, d).unbind(2))
    gq, gk, gv = (t.transpose(1, 2) for t in g.view(b, s, 3, h, d).unbind(2))
    near(dq, formula(gq, pos, f, False, 1.0, -1.0), gq)
    near(dk, formula(gk, pos, f, False, 1.0, -1.0), gk)
    assert torch.equal(dv, gv)
    y = x.detach().transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(cfa.fused_rotary_qkv(y, h, pos, f), want)
    wide = torch.zeros(b, s, 3 * h * d + 7, device=cuda, dtype=dtype)
    wide[..., 3:-4] = x.detach()
    assert torch.equal(cfa.fused_rotary_qkv(wide[..., 3:-4], h, pos, f), want)


def test_projection_into_attention(cuda):
    """fused_rotary_qkv into fused_attention_qkv, against the two plain formulas with torch's autograd."""
    b, s, h, d = 2, 65, 2, 64
    x = torch.randn(b, s, 3 * h * d, device=cuda, requires_grad=True)
    f, pos = cfa.rotary_frequencies(d, device=cuda), torch.arange(s, device=cuda)
    g = torch.randn(b, s, h * d, device=cuda)
    out = cfa.fused_attention_qkv(cfa.fused_rotary_qkv(x, h, pos, f), h, 0.125, True)
    (dx,) = torch.autograd.grad(out, x, g)
    y = x.detach().double().cpu().requires_grad_()
    q, k, v = (t.transpose(1, 2) for t in y.view(b, s, 3, h, d).unbind(2))
    a = pos.cpu().double()[:, None] * f.cpu()

    def turn(t):
        i, j = t[..., :32], t[..., 32:]
        return torch.cat((i * a.cos() - j * a.sin(), j * a.cos() + i * a.sin()), -1)

    w = torch.matmul(turn(q), turn(k).transpose(2, 3)) * 0.125
    w = torch.softmax(w.masked_fill(torch.ones(s, s, dtype=torch.bool).triu(1), -math.inf), -1)
    ref = torch.matmul(w, v).transpose(1, 2).reshape(b, s, h * d)
    (dref,) = torch.autograd.grad(ref, y, g.double().cpu())
    for got, want in ((out, ref), (dx, dref)):
        assert float((got.double().cpu() - want).norm() / want.norm()) <= 2e-6


def test_captured(cuda):
    q, k = operands(cuda, torch.float32, 2, 4, 2, 17, 64, seed=10)
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.zeros(2, 17, dtype=torch.int64, device=cuda)
    cfa.fused_rotary(q, k, pos, f)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cfa.fused_rotary(q, k, pos, f)
    for i in range(3):
        pos.random_(0, 10000), q.normal_()
        graph.replay()
        want = cfa.fused_rotary(q, k, pos, f)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty(cuda):
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.zeros(0, dtype=torch.int64, device=cuda)
    q, k = operands(cuda, torch.float32, 2, 4, 2, 0, 64)
    assert [list(y.shape) for y in cfa.fused_rotary(q, k, pos, f)] == [[2, 4, 0, 64], [2, 2, 0, 64]]


@pytest.mark.parametrize("scaling", [None, "linear", "base", "ramp"])
def test_scaled_frequencies(cuda, scaling):
    f = cfa.rotary_frequencies(64, scaling=scaling, factor=4.0, device=cuda)
    q, k = operands(cuda, torch.bfloat16, 1, 2, 2, 9, 64, seed=11)
    pos = torch.arange(70000, 70009, device=cuda)
    for x, y in zip((q, k), cfa.fused_rotary(q, k, pos, f, True)):
        near(y, formula(x, pos, f, True), x)


def test_far_operands(cuda):
    """Operands of more than 2^31 values: the last rows as those of a small call, bit for bit."""
    s = 1 << 22
    x = torch.empty(2, 1, s, 512, dtype=torch.float16, device=cuda)
    x[:, :, -5:] = torch.randn(2, 1, 5, 512, device=cuda).half()
    x[:, :, :5] = x[:, :, -5:]
    f, pos = cfa.rotary_frequencies(512, device=cuda), torch.arange(s, device=cuda) % (s - 5)
    y, z = cfa.fused_rotary(x, x, pos, f)
    want = cfa.fused_rotary(x[:, :, :5], x[:, :, :5], pos[:5], f)[0]
    for t in (y, z):
        assert torch.equal(t[:, :, :5], want) and torch.equal(t[:, :, -5:], want)


def test_impossible_heads_refused(cuda):
    qkv, f = torch.zeros(1, 2, 192, device=cuda), cfa.rotary_frequencies(64, device=cuda)
    for heads in (0, -1, 5, 65, (2 ** 64 - 1) // 3):
        with pytest.raises(cfa.FusedAttentionError, match="is not 3 x"):
            cfa.fused_rotary_qkv(qkv, heads, torch.arange(2, device=cuda), f)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [64, 10])
def test_in_place_through_the_c_abi(cuda, d, interleaved):
    """y may be x itself."""
    import ctypes

    from candle_fused_attn import _lib

    b, h, hk, s = 3, 5, 2, 70
    q, k = (t.contiguous() for t in operands(cuda, torch.float32, b, h, hk, s, d, seed=13))
    f, pos = cfa.rotary_frequencies(d, device=cuda), torch.arange(s, device=cuda)
    want = cfa.fused_rotary(q, k, pos, f, interleaved)
    at = (ctypes.c_void_p * 3)(q.data_ptr(), k.data_ptr(), None)
    st = _lib.arr([*q.stride()[:3], *k.stride()[:3], 0, 0, 0])
    _lib.check(_lib.lib().fattn_rotary(0, b, s, d, _lib.arr([h, hk, 0]), at, at, st, st, 0b11, pos.data_ptr(),
                                       64, _lib.arr([0, 1]), f.data_ptr(), d, int(interleaved), 1.0, 0,
                                       torch.cuda.current_stream().cuda_stream))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_training_captured(cuda):
    """A rotated projection's attention and its gradient, replayed with other values and positions, eager
    steps between: bit for bit the eager results."""
    b, s, h, d = 2, 50, 3, 64
    qkv = torch.randn(b, s, 3 * h * d, device=cuda, requires_grad=True)
    g, pos = torch.randn(b, s, h * d, device=cuda), torch.arange(s, device=cuda)
    f = cfa.rotary_frequencies(d, device=cuda)

    def step():
        out = cfa.fused_attention_qkv(cfa.fused_rotary_qkv(qkv, h, pos, f), h, 0.125, True)
        return [out.detach(), *torch.autograd.grad(out, qkv, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            qkv.normal_(), g.normal_(), pos.add_(1000 * i)
        graph.replay()
        out = [t.clone() for t in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_overlapping_views(cuda, dtype, interleaved):
    """Operands, projections and output gradients whose rows overlap (windows of a longer row: the stride
    of head_dim is another dimension's too): as of contiguous copies, bit for bit."""
    gen = torch.Generator().manual_seed(16)
    buf = torch.randn(4096, generator=gen).to(dtype).to(cuda)
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.arange(37, device=cuda)
    q = buf[:800].view(2, 4, 100).unfold(2, 64, 1)               # rows
    k = buf.as_strided((2, 3, 37, 64), (1000, 1, 20, 1), 3)      # heads
    x = buf.as_strided((2, 37, 3 * 64), (1000, 1, 1), 5)
    r = buf.as_strided((2, 37, 3 * 128), (1, 40, 1), 7)          # samples
    assert q.shape == (2, 4, 37, 64) and q.stride()[2:] == (1, 1)
    got = cfa.fused_rotary(q, k, pos, f, interleaved)
    want = cfa.fused_rotary(q.contiguous(), k.contiguous(), pos, f, interleaved)
    for a, b, t in zip(got, want, (q, k)):
        assert torch.equal(a, b)
        near(a, formula(t, pos, f, interleaved), t)
    for t, heads in ((x, 1), (r, 2)):
        assert torch.equal(cfa.fused_rotary_qkv(t, heads, pos, f, interleaved),
                           cfa.fused_rotary_qkv(t.contiguous(), heads, pos, f, interleaved))
    leaves = [t.contiguous().requires_grad_() for t in (q, k, x)]
    outs = [*cfa.fused_rotary(*leaves[:2], pos, f, interleaved),
            cfa.fused_rotary_qkv(leaves[2], 1, pos, f, interleaved)]
    grads = [torch.autograd.grad(outs, leaves, g, retain_graph=True)
             for g in ((q, k, x), (q.contiguous(), k.contiguous(), x.contiguous()))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_forward_mode_refused(cuda):
    """A tangent of an operand, or of the gradient that a backward is given."""
    import torch.autograd.forward_ad as forward_ad

    q, k = operands(cuda, torch.float32, 1, 2, 2, 5, 32, seed=14)
    f, pos = cfa.rotary_frequencies(32, device=cuda), torch.arange(5, device=cuda)
    x = torch.randn(1, 5, 3 * 64, device=cuda, requires_grad=True)
    leaves = [t.clone().requires_grad_() for t in (q, k)]
    outs = [*cfa.fused_rotary(*leaves, pos, f), cfa.fused_rotary_qkv(x, 2, pos, f)]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, k)
        with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
            cfa.fused_rotary(dual, k, pos, f)
        grads = [forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)) for y in outs]
        for y, leaf, g in zip(outs, (*leaves, x), grads):
            with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                torch.autograd.grad(y, leaf, g, retain_graph=True)
        with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
            torch.autograd.grad(outs[:2], leaves, grads[:2], retain_graph=True)
    for y, leaf in zip(outs, (*leaves, x)):
        assert torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)[0].shape == leaf.shape


def test_gradient_records_a_graph(cuda):
    """A gradient with a graph of it has one where the output's gradient does, and none where nothing in it
    can be differentiated (the rotation is linear)."""
    q, k = operands(cuda, torch.float32, 1, 2, 2, 5, 32, seed=15)
    f, pos = cfa.rotary_frequencies(32, device=cuda), torch.arange(5, device=cuda)
    q.requires_grad_()
    out = cfa.fused_rotary(q, k, pos, f)[0]
    for g in (torch.ones_like(out), torch.ones_like(out).requires_grad_()):
        (dq,) = torch.autograd.grad(out, q, g, create_graph=True)
        assert dq.requires_grad == g.requires_grad and (dq.grad_fn is not None) == g.requires_grad


def test_saved_tensors_elsewhere(cuda):
    """Positions and frequencies that the node saves may come back in other memory (activations kept on the
    host): the same gradients, bit for bit; of another type or shape: an error."""
    q, k = operands(cuda, torch.float32, 2, 4, 2, 9, 64, seed=17)
    gq, gk = operands(cuda, torch.float32, 2, 4, 2, 9, 64, seed=18)
    x, gx = (torch.randn(2, 9, 3 * 128, device=cuda) for _ in range(2))
    q, k, x = (t.detach().requires_grad_() for t in (q, k, x))
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.randint(0, 999, (9, 2), device=cuda).t()

    def step(context, two):
        with context:
            outs = cfa.fused_rotary(q, k, pos, f) if two else [cfa.fused_rotary_qkv(x, 2, pos, f)]
        return torch.autograd.grad(outs, (q, k) if two else x, (gq, gk) if two else gx)

    hooks = torch.autograd.graph.saved_tensors_hooks
    for two in (True, False):
        want = step(hooks(lambda t: t, lambda t: t), two)
        for context in (torch.autograd.graph.save_on_cpu(pin_memory=True), torch.autograd.graph.save_on_cpu(),
                        hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format))):
            assert all(torch.equal(a, b) for a, b in zip(step(context, two), want))
        for context in (hooks(lambda t: t, lambda t: t.float()), hooks(lambda t: t, lambda t: t[:1, :1]
                        if t.dim() == 2 else t), hooks(lambda t: t.cpu(), lambda t: t)):
            with pytest.raises(cfa.FusedAttentionError, match="fused_rotary"):
                step(context, two)
