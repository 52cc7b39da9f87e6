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
    # Few blocks and long walks: cut into chunks, with samples that fill some of them or none.
    (1, 2, 2, 130, 3000, 64, [2500]), (2, 16, 4, 100, 3000, 128, [3000, 10]), (1, 8, 1, 200, 600, 32, None),
    (2, 2, 1, 40, 2000, 64, [0, 1999]), (1, 16, 1, 500, 64, 64, None), (1, 1, 1, 1, 4000, 64, [3999]),
    (3, 1, 1, 2000, 1025, 32, [1025, 513, 256]),
    (256, 4, 2, 256, 40, 64, None), (171, 3, 1, 512, 33, 32, None),  # 64 queries per wave
    # Tiles of several heads in one workgroup, with lengths.
    (40, 6, 2, 33, 200, 64, [0, 77, 200, 31] * 10), (20, 10, 2, 65, 300, 32, [300, 0] * 10),
    (9, 12, 4, 97, 260, 128, None),
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


@pytest.mark.parametrize("b,h,hk,sq,sk,d,lengths", SHAPES)
def test_gradients(cuda, b, h, hk, sq, sk, d, lengths):
    q, k, v, g = operands(cuda, b, h, hk, sq, sk, d, seed=1)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    scale = d ** -0.5
    out = cfa.fused_cross_attention(q, k, v, scale, ints(cuda, lengths))
    got = torch.autograd.grad(out, leaves, g)
    exact = [t.detach().double().cpu().requires_grad_() for t in leaves]
    want = torch.autograd.grad(formula(*exact, scale, lengths), exact, g.double().cpu())
    # A sample that sees one key: dS = dP - D is 0 in exact arithmetic (D = dO.o, o = v), so dQ and dK have
    # no relative error there. Either sum of d products is off by at most d 2^-24 of the sum of their
    # magnitudes; dQ, dK by that twice, times the scale and a key's (for dK: the group's queries') values.
    seen = lengths or [sk] * b
    one = torch.tensor([n == 1 for n in seen])
    size = (g.double().cpu().abs().unflatten(1, (hk, -1)) @ exact[2].detach().abs()[:, :, None, 0, :, None])
    band = float(2 * d * 2.0 ** -24 * size.max() * scale)
    most = [band * float(exact[1].detach().abs().max()),
            band * (h // hk) * sq * float(exact[0].detach().abs().max())]
    for i, (x, ref) in enumerate(zip(got, want)):
        assert x.shape == ref.shape
        if i < 2 and bool(one.any()):
            assert float((x.double().cpu() - ref)[one].abs().max()) <= most[i]
            x, ref = x.cpu()[~one], ref[~one]
        assert x.numel() == 0 or rel(x, ref) <= TOL, "qkv"[i]
    for i, n in enumerate(lengths or []):
        assert float(got[1][i, :, n:].abs().sum() + got[2][i, :, n:].abs().sum()) == 0.0
        if n == 0:
            assert float(got[0][i].abs().max()) == 0.0
    again = torch.autograd.grad(cfa.fused_cross_attention(q, k, v, scale, ints(cuda, lengths)), leaves, g)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("sq,sk", [(3, 150), (200, 150), (200, 1500)])
def test_garbage_behind_the_last_key(cuda, sq, sk):
    """Infinities and NaN in keys that a sample does not see: no trace of them, their gradients 0."""
    q, k, v, g = operands(cuda, 3, 4, 2, sq, sk, 64, seed=2)
    lengths = [sk, 90, 0]
    bad_k, bad_v = k.clone(), v.clone()
    for i, n in enumerate(lengths):
        bad_k[i, :, n:], bad_v[i, :, n:] = float("nan"), float("inf")

    def run(k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = cfa.fused_cross_attention(*leaves, 0.125, ints(cuda, lengths))
        return [out, *torch.autograd.grad(out, leaves, g)]

    for x, y in zip(run(k, v), run(bad_k, bad_v)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("sq,sk", [(5, 70), (130, 70), (130, 1500)])
def test_non_finite_values_that_are_seen(cuda, sq, sk):
    """What the formula gives of an infinity among the values and a NaN among the queries, and nothing of
    them in other rows."""
    q, k, v, g = operands(cuda, 2, 2, 2, sq, sk, 64, seed=3)
    v[0, 0, 3, 5], q[1, 1, 2, 7] = float("inf"), float("nan")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cfa.fused_cross_attention(q, k, v, 0.125)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    exact = [t.detach().double().cpu().requires_grad_() for t in leaves]
    ref = formula(*exact, 0.125)
    want = [ref.detach(), *torch.autograd.grad(ref, exact, g.double().cpu())]
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, want):
        x = x.double().cpu()
        fine = y.isfinite()
        assert torch.equal(fine, x.isfinite()), name
        assert rel(x[fine], y[fine]) <= TOL, name


@pytest.mark.parametrize("sq,sk", [(5, 70), (5, 1500), (130, 70), (130, 1500)])
def test_scores_of_minus_infinity(cuda, sq, sk):
    """Keys that score minus infinity, whole tiles and chunks of them: no weight; a sample of nothing else:
    NaN, as the formula. (Positive queries, so that no infinite score is of another sign.)"""
    q, k, v, g = operands(cuda, 2, 2, 2, sq, sk, 64, seed=14)
    q = q.abs() + 0.5
    k[0, :, : sk * 2 // 3, 5] = -float("inf")
    k[1, 1, :, 5] = -float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cfa.fused_cross_attention(q, k, v, 0.125)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    exact = [t.detach().double().cpu().requires_grad_() for t in leaves]
    ref = formula(*exact, 0.125)
    want = [ref.detach(), *torch.autograd.grad(ref, exact, g.double().cpu())]
    assert bool(want[0][1, 1].isnan().all()) and bool(want[0][0].isfinite().all())
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, want):
        x = x.double().cpu()
        fine = y.isfinite()
        assert torch.equal(fine, x.isfinite()), name
        assert rel(x[fine], y[fine]) <= TOL, name


def test_strides_and_broadcasts(cuda):
    """Head views of fused projections, padded rows, odd offsets and broadcast keys: as contiguous ones."""
    b, h, sq, sk, d = 2, 4, 37, 50, 64
    kv = torch.randn(b, sk, 2, h, d, device=cuda)
    wide = torch.randn(b, h, sq, d + 4, device=cuda)
    odd = torch.randn(b * h * sq * d + 1, device=cuda)[1:].view(b, h, sq, d)
    g = torch.randn(b, h, sq, d, device=cuda)
    for q, k, v in ((wide[..., :d], kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)),
                    (odd, kv[:, :, 0, :1].transpose(1, 2).expand(b, h, sk, d),
                     kv[:1, :, 1].transpose(1, 2).expand(b, h, sk, d)),
                    (odd.permute(1, 0, 3, 2).contiguous().permute(1, 0, 3, 2), kv[:, :, 0].transpose(1, 2),
                     kv[:, :, 1].transpose(1, 2))):
        def run(q, k, v, g):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            out = cfa.fused_cross_attention(*leaves, 0.125)
            return [out, *torch.autograd.grad(out, leaves, g)]
        want = run(q.contiguous(), k.contiguous(), v.contiguous(), g)
        for gg in (g, g.transpose(1, 2).contiguous().transpose(1, 2),
                   torch.cat((g, g), -1)[..., :d]):
            for x, y in zip(run(q, k, v, gg), want):
                assert torch.equal(x, y)
    ge = g[:, :1, :1].expand_as(g)
    for x, y in zip(run(q, k, v, ge), run(q, k, v, ge.contiguous())):
        assert torch.equal(x, y)


def test_shared_heads_equal_repeated_ones(cuda):
    """A shared key head's gradient is the sum of its copies'."""
    q, k, v, g = operands(cuda, 2, 6, 2, 70, 90, 64, seed=4)  # (16 steps of a walk: not cut)
    a = [t.detach().requires_grad_() for t in (q, k, v)]
    b = [q.detach().requires_grad_(), *(t.repeat_interleave(3, 1).requires_grad_() for t in (k, v))]
    oa, ob = (cfa.fused_cross_attention(*x, 0.125) for x in (a, b))
    assert torch.equal(oa, ob)
    ga, gb = torch.autograd.grad(oa, a, g), torch.autograd.grad(ob, b, g)
    assert torch.equal(ga[0], gb[0])
    for x, y in zip(ga[1:], gb[1:]):
        assert rel(x, y.view(2, 2, 3, 90, 64).double().sum(2)) <= TOL


def test_gradient_against_differences(cuda):
    """Central differences of the fp64 formula in random directions, and the kernel's gradients."""
    q, k, v, g = operands(cuda, 1, 2, 1, 9, 40, 32, seed=5)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cfa.fused_cross_attention(q, k, v, 0.2, ints(cuda, [33])), leaves, g)
    x = [t.detach().double().cpu() for t in leaves]
    gen, e = torch.Generator().manual_seed(6), 1e-6
    for i in range(3):
        step = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        ends = []
        for s in (e, -e):
            y = list(x)
            y[i] = x[i] + s * step
            ends.append(float((formula(*y, 0.2, [33]) * g.double().cpu()).sum()))
        want = (ends[0] - ends[1]) / (2 * e)
        got = float((grads[i].double().cpu() * step).sum())
        # fp32: 2e-6 of the gradient's norm times the step's; the difference itself: 1e-15 / e and e^2.
        assert abs(got - want) <= TOL * float(grads[i].norm()) * float(step.norm()) + 1e-7


def test_some_gradients_only(cuda):
    q, k, v, g = operands(cuda, 2, 2, 2, 40, 50, 64, seed=7)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(cfa.fused_cross_attention(*leaves, 0.125), leaves, g)
    for i in range(3):
        x = [t.detach() for t in leaves]
        x[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(cfa.fused_cross_attention(*x, 0.125), x[i], g)[0], want[i])
    out = cfa.fused_cross_attention(*leaves, 0.125)
    (dq,) = torch.autograd.grad(out, q, g.requires_grad_(), create_graph=True)
    assert torch.equal(dq, want[0])
    with pytest.raises(RuntimeError, match="not differentiable"):
        dq.sum().backward()


def test_errors_of_a_backward(cuda):
    """What a backward refuses reaches the caller as the package's error or torch's own."""
    q, k, v, g = operands(cuda, 1, 2, 2, 20, 30, 64, seed=15)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cfa.fused_cross_attention(*leaves, 0.125)
    (dq,) = torch.autograd.grad(out, q, g, create_graph=True)
    with pytest.raises(cfa.FusedAttentionError, match="not differentiable"):
        dq.sum().backward()
    out = cfa.fused_cross_attention(*leaves, 0.125)
    torch.autograd.grad(out, q, g)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, q, g)
    x = q.detach().clone().requires_grad_() * 1.0
    out = cfa.fused_cross_attention(x, k, v, 0.125)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, k, g)


def test_threads(cuda):
    """Calls and their gradients from several threads at once: as one after the other."""
    import threading

    ops = [operands(cuda, 2, 4, 2, 3 + 40 * i, 300, 64, seed=16 + i) for i in range(4)]
    f, pos = cfa.rotary_frequencies(64, device=cuda), torch.arange(200, device=cuda)

    def step(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        a, b = cfa.fused_rotary(leaves[0], leaves[0] * 2.0, pos[: q.shape[2]], f)
        out = cfa.fused_cross_attention(a + b, leaves[1], leaves[2], 0.125)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want, got = [step(*x) for x in ops], [None] * 4
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [step(*ops[i]) for _ in range(10)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, ref in zip(got, want):
        assert all(torch.equal(x, y) for o in outs for x, y in zip(o, ref))


@pytest.mark.parametrize("shape", [(0, 2, 2, 5, 5), (2, 2, 2, 0, 5), (2, 2, 2, 5, 0), (2, 0, 0, 5, 5),
                                   (2, 2, 2, 0, 900), (2, 2, 2, 900, 0), (1, 2, 1, 900, 0)])
def test_empty(cuda, shape):
    q, k, v, g = operands(cuda, *shape, 64)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = cfa.fused_cross_attention(q, k, v, 0.125)
    assert out.shape == q.shape and float(out.abs().sum()) == 0.0
    for x, t in zip(torch.autograd.grad(out, leaves, g), leaves):
        assert x.shape == t.shape and float(x.abs().sum()) == 0.0


@pytest.mark.parametrize("sq", [1, 150])
def test_captured(cuda, sq):
    """Forward and backward replayed with other inputs and lengths in the same buffers, eager calls
    between: bit for bit the eager results."""
    q, k, v, g = operands(cuda, 2, 4, 2, sq, 900, 64, seed=8)
    lengths = ints(cuda, [900, 3])
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        out = cfa.fused_cross_attention(q, k, v, 0.125, lengths)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

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
            for t in (q, k, v, g):
                t.copy_(torch.randn_like(t))
            lengths.copy_(ints(cuda, [100 * i, 900 - 13 * i]))
        graph.replay()
        out = [t.clone() for t in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i


def test_side_streams(cuda):
    ops = [operands(cuda, 2, 4, 2, 1 + 99 * i, 700, 64, seed=9 + i) for i in range(2)]

    def step(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = cfa.fused_cross_attention(*leaves, 0.125)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = [step(*x) for x in ops]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*ops[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(outs, want[i]))


def test_equals_self_attention(cuda):
    """With keys of the queries' length and heads, what fused_attention gives."""
    q, k, v, g = operands(cuda, 3, 4, 4, 240, 240, 64, seed=12)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    res = []
    for f in (lambda: cfa.fused_cross_attention(q, k, v, 0.125),
              lambda: cfa.fused_attention(q, k, v, 0.125, False)):
        out = f()
        res.append([out.detach(), *torch.autograd.grad(out, leaves, g)])
    for x, y in zip(*res):
        assert rel(x, y) <= TOL


def test_decoder_layer(cuda):
    """The operators together: a decoder layer's attention in training (fused_rotary_qkv, causal
    fused_attention_qkv, fused_cross_attention to padded states), and the same layer token by token
    (paged_append, paged_attention, one query of fused_cross_attention): the same rows."""
    b, s, h, hk, d, sk = 2, 24, 4, 2, 64, 77
    lengths = ints(cuda, [77, 40])
    gen = torch.Generator(device=cuda).manual_seed(13)
    qkv = torch.randn(b, s, 3 * h * d, device=cuda, generator=gen, requires_grad=True)
    wq = (torch.randn(h * d, h * d, device=cuda, generator=gen) / (h * d) ** 0.5).requires_grad_()
    kv = torch.randn(b, sk, 2, hk, d, device=cuda, generator=gen, requires_grad=True)
    f = cfa.rotary_frequencies(d, device=cuda)

    def cross(x):
        q = (x @ wq).view(b, -1, h, d).transpose(1, 2)
        return cfa.fused_cross_attention(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), 0.125,
                                         lengths)

    mixed = cfa.fused_attention_qkv(
        cfa.fused_rotary_qkv(qkv, h, torch.arange(s, device=cuda), f), h, 0.125, True)
    want = cross(mixed)
    grads = torch.autograd.grad(want, (qkv, wq, kv), torch.ones_like(want))
    assert all(bool(x.isfinite().all()) and float(x.abs().max()) > 0 for x in grads)
    with torch.no_grad():
        kp, vp = (torch.zeros(6, h, 16, d, device=cuda) for _ in range(2))
        table = torch.tensor([[4, 1], [0, 5]], dtype=torch.int32, device=cuda)
        held = torch.zeros(b, dtype=torch.int32, device=cuda)
        for t in range(s):
            q, k, v = (x[:, t:t + 1].transpose(1, 2) for x in qkv.view(b, s, 3, h, d).unbind(2))
            q = cfa.paged_append(k, v, kp, vp, table, held, q=q, frequencies=f)
            held += 1
            x = cfa.paged_attention(q, kp, vp, table, held, 0.125)
            out = cross(x.transpose(1, 2).reshape(b, 1, h * d))
            # Two fp32 attentions and a product of 256 terms on either side.
            assert rel(out, want[:, :, t:t + 1]) <= 4 * TOL


@pytest.mark.parametrize("sq", [1, 150])
def test_forward_mode_refused(cuda, sq):
    """A tangent of an operand, or of the gradient that the backward is given."""
    import torch.autograd.forward_ad as forward_ad

    q, k, v, g = operands(cuda, 1, 2, 2, sq, 30, 64, seed=20)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = cfa.fused_cross_attention(*leaves, 0.125)
    with forward_ad.dual_level():
        for i in range(3):
            x = [q, k, v]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                cfa.fused_cross_attention(*x, 0.125)
        with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
            torch.autograd.grad(out, leaves, forward_ad.make_dual(g, g))


@pytest.mark.parametrize("sq", [1, 150])
def test_far_keys(cuda, sq):
    """Samples more than 2^31 values apart: as contiguous ones, bit for bit, gradients too."""
    b, h, sk, d = 2, 2, 70, 64
    q, k, v, g = operands(cuda, b, h, h, sq, sk, d, seed=21)
    k, v = (t.contiguous() for t in (k, v))
    far = torch.empty(2 ** 31 + 2 ** 16, device=cuda)
    at = [far.as_strided(k.shape, (2 ** 31 + 64, sk * d, d, 1), i * h * sk * d) for i in range(2)]
    at[0].copy_(k), at[1].copy_(v)
    out = []
    for x in ((q, k, v), (q, *at)):
        leaves = [t.detach().requires_grad_() for t in x]
        o = cfa.fused_cross_attention(*leaves, 0.125, ints(cuda, [70, 33]))
        out.append([o.detach(), *torch.autograd.grad(o, leaves, g)])
    assert all(torch.equal(x, y) for x, y in zip(*out))
    assert bool(out[0][0].isfinite().all()) and float(out[0][0].abs().max()) > 0


@pytest.mark.parametrize("sq,sk,lengths", [(1, 300, None), (40, 70, [70, 3]), (150, 600, None)])
def test_saved_tensors_elsewhere(cuda, sq, sk, lengths):
    """What the node saves may come back in other memory and another layout (activations kept on the host):
    the same gradients, bit for bit; of another type or shape: an error."""
    q, k, v, g = operands(cuda, 2, 4, 2, sq, sk, 64, seed=22)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    n = ints(cuda, lengths)

    def step(context):
        with context:
            out = cfa.fused_cross_attention(q, k, v, 0.125, n)
        return torch.autograd.grad(out, (q, k, v), g)

    hooks = torch.autograd.graph.saved_tensors_hooks
    want = step(hooks(lambda t: t, lambda t: t))
    for context in (torch.autograd.graph.save_on_cpu(pin_memory=True), torch.autograd.graph.save_on_cpu(),
                    hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)),
                    hooks(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1))):
        assert all(torch.equal(x, y) for x, y in zip(step(context), want))
    for context in (hooks(lambda t: t, lambda t: t.half() if t.is_floating_point() else t),
                    hooks(lambda t: t, lambda t: t[..., :-1] if t.dim() == 3 else t),
                    hooks(lambda t: t, lambda t: t[:1]),
                    hooks(lambda t: t.cpu(), lambda t: t)):
        with pytest.raises(cfa.FusedAttentionError, match="fused_cross_attention: "):
            step(context)
