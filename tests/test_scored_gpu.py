"""Attention of capped, biased and masked scores on the GPU, forward and backward, against the formula in 64
bits and its differentiation: documents that begin and end inside tiles, in and out of order, padding, rows
that see nothing, prefixes, queries that are the last of a longer context, shared key heads, caps that all
or no scores come near, values that are not finite in places that are and are not seen, strides.

Tolerances. 2e-6 normwise of each (batch, head)'s output and gradients, the bar of every fp32 attention test
here. A score y of a cap or of slopes carries besides 5 x 2^-24 of |y| (x / cap, tanh to 1.3 x 2^-24, the
product and the difference), which is a weight's relative error, over the keys that weigh anything; the
derivative 1 - tanh^2 loses 4 x 2^-24 of 1 where it is itself of that size, so no more than the weights do."""
from __future__ import annotations

import math

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu


def operands(b, h, hk, sq, sk, d, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    q, g = (torch.randn(b, h, sq, d, generator=gen) for _ in range(2))
    k, v = (torch.randn(b, hk, sk, d, generator=gen) for _ in range(2))
    return q * spread, k, v, g


def visible(b, sq, sk, causal, documents=None, prefix=None):
    j = torch.arange(sk)
    i = j[sk - sq:]
    seen = torch.ones(b, sq, sk, dtype=torch.bool)
    if causal:
        seen = (j[None, :] <= i[:, None]).expand(b, sq, sk)
        if prefix is not None:
            seen = seen | (j < prefix.clamp(0, sk)[:, None, None])
    if documents is not None:
        mine = documents[:, sk - sq:, None]
        seen = seen & (documents[:, None] == mine) & (mine >= 0)
    return seen


def formula(q, k, v, g, scale, causal, cap=None, slopes=None, documents=None, prefix=None):
    """Output and gradients in 64 bits, and the largest |y| of a key that weighs 1e-3 of its row's heaviest."""
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    q, k, v = (t.double().requires_grad_(True) for t in (q, k, v))
    seen = visible(b, sq, sk, causal, documents, prefix)[:, None]
    empty = ~seen.any(-1, keepdim=True)
    kk, vv = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    y = torch.matmul(q, kk.transpose(2, 3)) * scale
    if cap is not None:
        y = cap * torch.tanh(y / cap)
    if slopes is not None:
        j = torch.arange(sk, dtype=torch.float64)
        y = y - slopes.double().cpu()[:, None, None] * (j[sk - sq:, None] - j).abs()
    p = torch.softmax(y.masked_fill(~seen & ~empty, -math.inf), -1).masked_fill(empty, 0.0)
    top = 0.0
    if cap is not None or slopes is not None:
        heavy = seen & (p > 1e-3 * p.amax(-1, keepdim=True))
        top = float(y.detach()[heavy].abs().max()) if bool(heavy.any()) else 0.0
    o = torch.matmul(p, vv)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), g.double())], top


def run(dev, q, k, v, g, *args, **how):
    q, k, v = (t.to(dev).requires_grad_(True) for t in (q, k, v))
    how = {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    out = cfa.fused_scored_attention(q, k, v, *args, **how)
    return [out.detach(), *torch.autograd.grad(out, (q, k, v), g.to(dev))]


def check(got, ref, top=0.0, steep=0.0):
    """Each (batch, head)'s error over its norm, or over 1e-3 of the tensor's largest head (a head of few
    visible pairs may have next to no gradient). steep: a gradient's relative error besides."""
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, ref):
        x = x.double().cpu()
        assert x.shape == y.shape and bool(x.isfinite().all()), name
        n = y.flatten(2).norm(dim=-1)
        err = (x - y).flatten(2).norm(dim=-1) / n.clamp_min(max(1e-3 * float(n.max()), 1e-30))
        bar = 2e-6 + 5 * 2.0 ** -24 * top + (0.0 if name == "o" else steep)
        assert float(err.max()) <= bar, (name, float(err.max()), bar)


def ids_of(spans, sk):
    """Documents of these lengths one after the other; what they leave of sk is padding."""
    out = torch.full((len(spans), sk), -1, dtype=torch.int32)
    for row, lengths in zip(out, spans):
        at = 0
        for n, m in enumerate(lengths):
            row[at:at + m] = n
            at += m
    return out


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 1, 33, 33), (1, 4, 2, 130, 130), (2, 6, 2, 200, 333), (1, 2, 2, 5, 700),
          (3, 3, 3, 64, 64), (1, 2, 1, 1, 1500)]


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("kind", ["plain", "capped", "slopes", "both"])
def test_shapes_and_scores(cuda, shape, d, causal, kind):
    b, h, hk, sq, sk = shape
    cap = 4.0 if kind in ("capped", "both") else None
    slopes = torch.linspace(0.01, 1.0, h) if kind in ("slopes", "both") else None
    q, k, v, g = operands(b, h, hk, sq, sk, d, seed=sk + d, spread=2.0 if cap else 1.0)
    if kind != "plain" and sk == 1:
        pytest.skip("a query that sees one key has no gradient")
    args = (d ** -0.5, causal)
    ref, top = formula(q, k, v, g, *args, cap=cap, slopes=slopes)
    got = run(cuda, q, k, v, g, *args, cap=cap, slopes=slopes)
    if sk == 1:
        assert all(float(x.abs().max()) <= 1e-5 for x in got[1:3])
        got, ref = [got[0], got[3]], [ref[0], ref[3]]
    check(got, ref, top)
    again = run(cuda, q, k, v, g, *args, cap=cap, slopes=slopes)
    assert all(torch.equal(x, y) for x, y in zip(got, again[:1] + again[-1:] if sk == 1 else again))


DOCUMENTS = {
    "packed": [[100, 31, 1, 64, 104], [300], [1] * 40 + [2] * 60 + [150 - 10]],
    "padded": [[50, 70], [299], [0]],
    "tiles": [[32, 64, 96, 108], [128, 128, 44], [31, 33, 31, 33, 172]],
}


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("kind", DOCUMENTS)
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("sq", [300, 77])
@pytest.mark.parametrize("scores", [False, True], ids=["plain", "both"])
def test_documents(cuda, kind, d, causal, sq, scores):
    ids = ids_of(DOCUMENTS[kind], 300)
    q, k, v, g = operands(3, 4, 2, sq, 300, d, seed=1)
    how = dict(documents=ids)
    if scores:
        how.update(cap=2.0, slopes=torch.tensor([0.0, 0.1, -0.02, 0.7]))
    ref, top = formula(q, k, v, g, d ** -0.5, causal, **how)
    got = run(cuda, q, k, v, g, d ** -0.5, causal, **how)
    check(got, ref, top)
    empty = ~visible(3, sq, 300, causal, ids).any(-1)
    assert float(got[0].cpu().transpose(1, 2)[empty].abs().sum()) == 0.0
    assert float(got[1].cpu().transpose(1, 2)[empty].abs().sum()) == 0.0
    unseen = ~visible(3, sq, 300, causal, ids).any(1)
    assert float(got[2].cpu().transpose(1, 2)[unseen].abs().sum()) == 0.0
    assert float(got[3].cpu().transpose(1, 2)[unseen].abs().sum()) == 0.0


@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_documents_in_any_order(cuda, causal):
    """Ids that come back, interleaved ids, large ones, the least and largest of their type."""
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(-1, 4, (4, 500), generator=gen, dtype=torch.int32)
    ids[1] = ids[1] * 1000000007 % 2 ** 31
    ids[2] = torch.where(ids[2] > 1, 2 ** 31 - 1, -2 ** 31)
    ids[3] = torch.arange(500) // 40 % 3
    q, k, v, g = operands(4, 2, 1, 500, 500, 64, seed=3)
    ref, top = formula(q, k, v, g, 0.125, causal, documents=ids)
    check(run(cuda, q, k, v, g, 0.125, causal, documents=ids), ref, top)


@pytest.mark.parametrize("sq", [400, 90])
def test_prefixes(cuda, sq):
    """None, all, a part that ends inside and at a tile, past both ends of the sample; with documents too."""
    prefix = torch.tensor([0, 400, 77, 128, -5, 1000, 1], dtype=torch.int32)
    q, k, v, g = operands(7, 2, 2, sq, 400, 64, seed=4)
    ids = ids_of([[150, 200, 30]] * 7, 400)
    for how in (dict(prefix=prefix), dict(prefix=prefix, documents=ids),
                dict(prefix=prefix, slopes=torch.tensor([0.02, 0.3]))):
        ref, top = formula(q, k, v, g, 0.125, True, **how)
        check(run(cuda, q, k, v, g, 0.125, True, **how), ref, top)


@pytest.mark.parametrize("cap,spread", [(0.05, 1.0), (0.5, 30.0), (30.0, 1.0), (50.0, 20.0), (1e4, 1.0)])
def test_caps(cuda, cap, spread):
    """All scores far past the cap, some, none near it. A score in 32 bits carries 2^-23 of the scores' size
    (sums of 64 products: 1e-7 normwise; the size is `spread`), so x / cap carries 2^-23 spread / cap, and
    1 - tanh^2, whose logarithm has a slope of 2 at most, twice that of itself: a gradient's error besides."""
    q, k, v, g = operands(2, 2, 2, 150, 150, 64, seed=5, spread=spread)
    ref, top = formula(q, k, v, g, 0.125, True, cap=cap)
    got = run(cuda, q, k, v, g, 0.125, True, cap=cap)
    check(got, ref, top, 2 * 2.0 ** -23 * spread / cap)


@pytest.mark.parametrize("causal,prefix", [(True, None), (True, [90, 400]), (False, None)], ids=["causal", "prefix", "all"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_steep_slopes(cuda, d, causal, prefix):
    """Slopes under which only a key's next neighbours weigh: as exact as gentle ones, whose distances are sums."""
    slopes = torch.tensor([0.6, 0.8, 3.0, 17.0, 300.0, -0.9, 1e6, 0.7])
    q, k, v, g = operands(2, 8, 4, 400, 400, d, seed=22)
    how = dict(slopes=slopes, prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32))
    got = run(cuda, q, k, v, g, d ** -0.5, causal, **how)
    ref, _ = formula(q, k, v, g, d ** -0.5, causal, **how)
    # O and dV, head by head: |y| of a key that weighs 1e-3 is that of the scores and 7 more, but for the head of
    # slope -0.9, where it is 0.9 x 400 (the third of the four key heads has it too).
    for i, keep in ((0, [0, 1, 2, 3, 4, 6, 7]), (3, [0, 1, 3])):
        check([got[i][:, keep].contiguous()], [ref[i][:, keep]], 12.0)
    check([got[0]], [ref[0]], 0.9 * 400)
    check([got[3]], [ref[3]], 0.9 * 400)
    # dQ and dK beside the largest head's: where one key has all the weight, dS = P (dP - D) is the difference of
    # two sums that are as large as where it has not, and carries their errors, 2e-6 of these, alone.
    for x, y in zip(got[1:3], ref[1:3]):
        n = y.flatten(2).norm(dim=-1).max()
        err = (x.double().cpu() - y).flatten(2).norm(dim=-1) / n
        assert float(err.max()) <= 2e-6 + 5 * 2.0 ** -24 * 0.9 * 400, float(err.max())


def test_equals_plain_attention(cuda):
    """Without any of the forms: fused_attention's and fused_cross_attention's results, to rounding."""
    q, k, v, g = operands(2, 4, 4, 300, 300, 64, seed=6)
    for causal in (False, True):
        got = run(cuda, q, k, v, g, 0.125, causal)
        x = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
        out = cfa.fused_attention(*x, 0.125, causal)
        check(got, [t.double().cpu() for t in (out.detach(), *torch.autograd.grad(out, x, g.to(cuda)))])


def test_large_scores_and_sinks(cuda):
    """Scores to +-100 in an order that moves the reference, a negative scale, one key of all the weight."""
    q, k, v, g = operands(1, 2, 2, 260, 260, 64, seed=7)
    q, k = q * torch.linspace(0.1, 8, 260)[:, None], k * torch.linspace(3, 0.2, 260)[:, None]
    k[:, :, 130] *= 6
    for scale in (0.3, -0.3):
        for how in (dict(), dict(slopes=torch.tensor([0.05, 1.5]))):
            ref, _ = formula(q, k, v, g, scale, True, **how)
            got = run(cuda, q, k, v, g, scale, True, **how)
            # (Scores of up to S carry 2^-23 S in 32 bits, whatever forms them: here 200.)
            check(got, ref, 200.0)


# --- Values that are not finite --------------------------------------------------------------------


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), 3e38])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_hidden_values_leave_no_trace(cuda, bad, causal):
    """In padding, in other documents and after the last query's position: what is not seen."""
    ids = ids_of([[60, 60, 50], [170]], 200)
    q, k, v, g = operands(2, 2, 1, 200, 200, 64, seed=8)
    clean = run(cuda, q, k, v, g, 0.125, causal, documents=ids, cap=5.0)
    q2, k2, v2, g2 = (t.clone() for t in (q, k, v, g))
    for t in (q2, k2, v2, g2):
        t[:, :, 170:] = bad
    got = run(cuda, q2, k2, v2, g2, 0.125, causal, documents=ids, cap=5.0)
    check([t.cpu() for t in got], [t.double().cpu() for t in clean])
    # One document's values: the others' results, bit for bit or by the fp32 path.
    for t in (q2, k2, v2, g2):
        t[:, :, 170:] = 0.0
        t[0, :, 60:120, 5] = bad
    got = run(cuda, q2, k2, v2, g2, 0.125, causal, documents=ids, cap=5.0)
    for x, y in zip(got, clean):
        for rows in (slice(0, 60), slice(120, 200)):
            a, e = x[0, :, rows].double(), y[0, :, rows].double()
            assert bool(a.isfinite().all())
            assert float((a - e).norm() / e.norm()) <= 2e-6


def test_seen_values_give_what_the_formula_gives(cuda):
    """NaN and infinities that are seen: not finite where the formula is not, its values elsewhere."""
    for bad in (float("nan"), float("inf")):
        q, k, v, g = operands(1, 2, 2, 150, 150, 64, seed=9)
        v[0, 0, 40, 3] = bad
        k[0, 1, 90, 7] = bad
        # (The formula over the seen keys alone: a product with a weight of 0 would bring in the others.)
        seen = visible(1, 150, 150, True)[:, None]
        y = torch.matmul(q.double(), k.double().transpose(2, 3)) * 0.125
        p = torch.softmax(y.masked_fill(~seen, -math.inf), -1)
        e = (p[..., None] * v.double()[:, :, None]).masked_fill(~seen[..., None], 0.0).sum(-2)
        got = run(cuda, q, k, v, g, 0.125, True)
        o = got[0].double().cpu()
        assert torch.equal(o.isfinite(), e.isfinite())
        fine = e.isfinite()
        assert float((o - e)[fine].norm() / e[fine].norm()) <= 2e-6


@pytest.mark.parametrize("sk", [70, 1500])
def test_infinite_scores_within_a_cap(cuda, sk):
    """A cap makes weights of infinite scores; scores of minus infinity throughout are NaN without one, and
    rows that see nothing stay 0 beside them. Whole walks and chunks of them."""
    q, k, v, _ = operands(1, 1, 1, 3, sk, 64, seed=10)
    k[0, 0, 5, 0] = float("inf")
    q[0, 0, :, 0] = torch.tensor([1.0, -1.0, 0.5])
    ref, top = formula(q, k, v, torch.zeros_like(q), 0.125, False, cap=3.0)
    out = cfa.fused_scored_attention(*(t.to(cuda) for t in (q, k, v)), 0.125, False, cap=3.0)
    assert float((out.double().cpu() - ref[0]).norm() / ref[0].norm()) <= 2e-6 + 5 * 2.0 ** -24 * top
    q, k = torch.zeros(1, 1, 3, 64), torch.zeros(1, 1, sk, 64)
    q[..., 0], k[..., 0] = 1.0, -float("inf")
    ids = torch.zeros(1, sk, dtype=torch.int32)
    ids[0, -1] = -1
    out = cfa.fused_scored_attention(q.to(cuda), k.to(cuda), v.to(cuda), 0.125, False, documents=ids.to(cuda))
    assert bool(out[0, 0, :2].isnan().all()) and float(out[0, 0, 2].abs().max()) == 0.0


# --- Operands, gradients, streams ------------------------------------------------------------------


def test_strides_and_broadcasts(cuda):
    b, h, hk, s, d = 2, 4, 2, 100, 64
    q, k, v, g = operands(b, h, hk, s, s, d, seed=11)
    ids = ids_of([[40, 60], [100]], s)
    want = run(cuda, q, k, v, g, 0.125, True, documents=ids)
    wide = torch.zeros(b, 2 * s, dtype=torch.int32)
    wide[:, 7:7 + s] = ids
    for make in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.nn.functional.pad(t, (1, 3))[..., 1:1 + d],
                 lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        x = [make(t).to(cuda).requires_grad_(True) for t in (q, k, v)]
        out = cfa.fused_scored_attention(*x, 0.125, True, documents=wide.to(cuda)[:, 7:7 + s])
        got = [out.detach(), *torch.autograd.grad(out, x, make(g).to(cuda))]
        assert all(torch.equal(a, e) for a, e in zip(got, want))
    one = k[:, :1].to(cuda).requires_grad_(True)
    shared = one.expand(b, hk, s, d)
    out = cfa.fused_scored_attention(q.to(cuda), shared, v.to(cuda), 0.125, True)
    (dk,) = torch.autograd.grad(out.sum(), one)
    kk = shared.detach().clone().requires_grad_(True)
    out = cfa.fused_scored_attention(q.to(cuda), kk, v.to(cuda), 0.125, True)
    (each,) = torch.autograd.grad(out.sum(), kk)
    assert float((dk - each.sum(1, keepdim=True)).norm() / dk.norm()) <= 1e-6
    (gq,) = torch.autograd.grad(cfa.fused_scored_attention(
        x[0], x[1].detach(), x[2].detach(), 0.125, True, documents=ids.to(cuda)).sum(), x[0])
    assert gq.shape == q.shape


def test_gradient_against_differences(cuda):
    """The change of a weighed sum of the output along a direction, by central differences in 64 bits of the
    formula and by the gradients."""
    q, k, v, g = operands(1, 4, 2, 70, 90, 32, seed=12, spread=2.0)
    how = dict(cap=3.0, slopes=torch.tensor([0.1, 0.2, 0.0, -0.1]), documents=ids_of([[30, 60]], 90),
               prefix=torch.tensor([50], dtype=torch.int32))
    got = run(cuda, q, k, v, g, 0.2, True, **how)
    gen = torch.Generator().manual_seed(13)
    for i, x in enumerate((q, k, v)):
        way = torch.randn(x.shape, generator=gen)
        ends = []
        for step in (1e-4, -1e-4):
            moved = [t.double() + (step * way.double() if n == i else 0) for n, t in enumerate((q, k, v))]
            ends.append(float((formula(*moved, g, 0.2, True, **how)[0][0] * g.double()).sum()))
        slope = (ends[0] - ends[1]) / 2e-4
        mine = float((got[1 + i].double().cpu() * way.double()).sum())
        # (A difference's own error is of 1e-8 of the second derivative's size, the gradient's 2e-6 of its norm.)
        assert abs(mine - slope) <= 3e-6 * float(got[1 + i].norm()) * float(way.norm()), (i, mine, slope)


@pytest.mark.parametrize("sq", [150, 3])
def test_captured(cuda, sq):
    """Forward and backward in a graph, replayed on other inputs, ids and prefixes in the same buffers."""
    q, k, v, g = (t.to(cuda) for t in operands(2, 4, 2, sq, 1000 if sq == 3 else sq, 64, seed=14))
    sk = k.shape[2]
    ids, prefix = torch.zeros(2, sk, dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4], device=cuda)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = cfa.fused_scored_attention(*leaves, 0.125, True, cap=5.0, slopes=slopes, documents=ids, prefix=prefix)
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
            ids.copy_(torch.arange(sk, device=cuda) * (i + 1) // sk)
            prefix.fill_(17 * i)
        graph.replay()
        out = [t.clone() for t in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), i


@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_chunks(cuda, d):
    """Few rows over many keys: walks in a hundred chunks, many of which a row does not see at all."""
    sk = 40000 if d == 64 else 20000
    q, k, v, g = operands(1, 2, 1, 5, sk, d, seed=21)
    ids = ids_of([[sk // 7] * 6 + [sk - 6 * (sk // 7) - 2]], sk)
    for how in ({}, {"documents": ids}, {"documents": ids, "prefix": torch.tensor([sk - 9], dtype=torch.int32)}):
        got = run(cuda, q, k, v, g, d ** -0.5, True, cap=9.0, **how)
        ref, top = formula(q, k, v, g, d ** -0.5, True, cap=9.0, **how)
        check(got, ref, top)


def test_side_streams(cuda):
    """Two calls in flight, each with its own workspace (chunks of a long walk)."""
    cases = [[t.to(cuda) for t in operands(1, 2, 2, 5, 4000, 64, seed=15 + i)] for i in range(2)]
    want = [cfa.fused_scored_attention(*c[:3], 0.125, True, cap=4.0) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cfa.fused_scored_attention(*cases[i][:3], 0.125, True, cap=4.0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


@pytest.mark.parametrize("shape", [(0, 2, 2, 3, 3), (2, 0, 0, 3, 3), (2, 2, 2, 0, 3), (2, 2, 2, 0, 0)])
def test_empty(cuda, shape):
    b, h, hk, sq, sk = shape
    q, k, v, g = operands(b, h, hk, sq, sk, 64)
    got = run(cuda, q, k, v, g, 0.125, True)
    assert [t.shape for t in got] == [q.shape, q.shape, k.shape, v.shape]
    assert all(float(t.abs().sum()) == 0.0 for t in got)


def test_far_rows(cuda):
    """Samples 2^31 values apart."""
    far = torch.empty(2, 2 ** 31 // 64 + 64, 64, device=cuda)
    q, k, v, g = operands(2, 1, 1, 40, 40, 64, seed=16)
    views = []
    for t in (q, k, v):
        x = far[:, len(views) * 40:][:, :40][:, None]
        x.copy_(t)
        views.append(x.requires_grad_(False))
    out = cfa.fused_scored_attention(*views, 0.125, True)
    assert torch.equal(out, cfa.fused_scored_attention(*(t.to(cuda) for t in (q, k, v)), 0.125, True))


def test_some_gradients_alone(cuda):
    """Gradients of q alone, and with frozen keys and values: those of the full call."""
    q, k, v, g = (t.to(cuda) for t in operands(2, 4, 2, 130, 200, 64, seed=24))
    how = dict(cap=4.0, slopes=torch.tensor([0.1, 0.2, 0.3, 0.4], device=cuda))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    full = torch.autograd.grad(cfa.fused_scored_attention(*leaves, 0.125, True, **how), leaves, g)
    x = q.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(cfa.fused_scored_attention(x, k, v, 0.125, True, **how), x, g)[0], full[0])
    x = v.clone().requires_grad_(True)
    cfa.fused_scored_attention(q, k, x, 0.125, True, **how).backward(g)
    assert torch.equal(x.grad, full[2])
    # One tensor as keys and values: the sum of both gradients.
    x = k.clone().requires_grad_(True)
    y = [k.clone().requires_grad_(True) for _ in range(2)]
    one = torch.autograd.grad(cfa.fused_scored_attention(q, x, x, 0.125, True, **how), x, g)[0]
    two = torch.autograd.grad(cfa.fused_scored_attention(q, *y, 0.125, True, **how), y, g)
    assert torch.equal(one, two[0] + two[1])


def test_far_positions(cuda):
    """Positions past 2^24, which are no floats: their distances are those of near ones."""
    sk, near = 2 ** 24 + 77, 3000
    q, k, v, g = operands(1, 2, 1, 40, near, 32, seed=23)
    far = [torch.zeros(1, 1, sk, 32, device=cuda) for _ in range(2)]
    for x, y in zip(far, (k, v)):
        x[:, :, -near:] = y.to(cuda)
    slopes = torch.tensor([0.05, 0.3])  # (a key 3000 away weighs e^-150)
    leaves = [t.requires_grad_(True) for t in (q.to(cuda), *far)]
    out = cfa.fused_scored_attention(*leaves, 0.2, True, slopes=slopes.to(cuda))
    dq, dk, dv = torch.autograd.grad(out, leaves, g.to(cuda))
    ref, top = formula(q, k, v, g, 0.2, True, slopes=slopes)
    check([out.detach(), dq, dk[:, :, -near:], dv[:, :, -near:]], ref, top)
    assert float(dk[:, :, :-near].abs().max()) == 0.0 and float(dv[:, :, :-near].abs().max()) < 1e-30


def test_saved_tensors_elsewhere(cuda):
    """Activations kept on the host between the forward and the backward, which come back contiguous."""
    q, k, v, g = operands(2, 4, 2, 100, 100, 64, seed=17)
    ids = ids_of([[40, 60], [90]], 100)
    want = run(cuda, q, k, v, g, 0.125, True, documents=ids, prefix=torch.tensor([3, 60], dtype=torch.int32))
    with torch.autograd.graph.save_on_cpu():
        x = [t.transpose(1, 2).contiguous().transpose(1, 2).to(cuda).requires_grad_(True) for t in (q, k, v)]
        out = cfa.fused_scored_attention(*x, 0.125, True, documents=ids.to(cuda),
                                         prefix=torch.tensor([3, 60], dtype=torch.int32, device=cuda))
    got = [out.detach(), *torch.autograd.grad(out, x, g.to(cuda))]
    assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_refusals_on_the_device(cuda):
    q, k, v, _ = (t.to(cuda) for t in operands(2, 4, 2, 10, 10, 64))
    ids, slopes = torch.zeros(2, 10, dtype=torch.int32, device=cuda), torch.zeros(4, device=cuda)
    call = lambda *x, **how: cfa.fused_scored_attention(*x, 0.125, True, **how)
    for fn, text in [
        (lambda: call(torch.cat((q, q), 2), k, v), "sq <= sk"),
        (lambda: call(q, k, v[:, :1]), "expected"),
        (lambda: call(q[:, :3], k, v), "no multiple"),
        (lambda: call(q[..., :48], k[..., :48], v[..., :48]), "got 48"),
        (lambda: call(q.half(), k, v), "must be float32"),
        (lambda: call(q, k, v, cap=0.0), "a cap from"),
        (lambda: call(q, k, v, cap=1e31), "a cap from"),
        (lambda: call(q, k, v, slopes=slopes[:2]), "slopes \\[4\\]"),
        (lambda: call(q, k, v, slopes=slopes.requires_grad_()), "no gradient of the slopes"),
        (lambda: call(q, k, v, documents=ids[:, :9]), "documents"),
        (lambda: call(q, k, v, documents=ids.long()), "int32"),
        (lambda: call(q, k, v, documents=ids.t().contiguous().t()), "contiguous rows"),
        (lambda: call(q, k, v, documents=ids.cpu()), "HIP device"),
        (lambda: call(q, k, v, prefix=ids[0]), "prefix"),
    ]:
        with pytest.raises(cfa.FusedAttentionError, match=text):
            fn()
    x = q.clone().requires_grad_(True)
    out = call(x, k, v)
    (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(cfa.FusedAttentionError, match="not differentiable"):
        g.sum().backward()


# --- Together ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["f32", "fp4"])
def test_trained_and_served_alike(cuda, cache):
    """A decoder layer's attention with a cap and slopes: a prompt whole, the prompt in two chunks (the second
    over what paged_read brings back), and token by token over the cache, give the same outputs."""
    b, h, hk, s, d, page = 2, 4, 2, 75, 64, 16
    gen = torch.Generator().manual_seed(18)
    q, k, v = (torch.randn(b, n, s, d, generator=gen).to(cuda) for n in (h, hk, hk))
    f, pos = cfa.rotary_frequencies(d, device=cuda), torch.arange(s, device=cuda)
    how = dict(cap=6.0, slopes=torch.tensor([0.5, 0.1, 0.02, 0.0], device=cuda))
    wide, kind = (cfa.fp4_row_bytes(d), torch.uint8) if cache == "fp4" else (d, torch.float32)
    kp, vp = (torch.zeros(2 * 5, hk, page, wide, dtype=kind, device=cuda) for _ in range(2))
    table = torch.arange(10, dtype=torch.int32, device=cuda).view(2, 5)
    lengths = torch.zeros(b, dtype=torch.int32, device=cuda)
    qt, kt = cfa.fused_rotary(q, k, pos, f)
    if cache == "fp4":  # (what the cache will hold of them)
        cfa.paged_append(k, v, kp, vp, table, lengths, frequencies=f)
        kt, v = cfa.paged_read(kp, vp, table, lengths + s, s, dtype=torch.float32)
        v0 = v
        kp.zero_(), vp.zero_()
    else:
        v0 = v
    whole = cfa.fused_scored_attention(qt, kt, v, 0.125, True, **how)
    n = 40
    cfa.paged_append(k[:, :, :n], v0[:, :, :n], kp, vp, table, lengths, frequencies=f)
    lengths += n
    first = cfa.fused_scored_attention(qt[:, :, :n], *cfa.paged_read(kp, vp, table, lengths, n, dtype=torch.float32),
                                       0.125, True, **how)
    cfa.paged_append(k[:, :, n:], v0[:, :, n:], kp, vp, table, lengths, frequencies=f)
    lengths += s - n
    kr, vr = cfa.paged_read(kp, vp, table, lengths, s, dtype=torch.float32)
    assert torch.equal(kr, kt) and torch.equal(vr, v)
    second = cfa.fused_scored_attention(qt[:, :, n:], kr, vr, 0.125, True, **how)
    bar = 4e-6 + 10 * 2.0 ** -24 * 6.0  # (of two results)
    rel = lambda x, y: float(((x - y).norm(dim=-1) / y.norm(dim=-1)).max())
    assert rel(torch.cat((first, second), 2), whole) <= bar
    for t in (0, 1, 39, 40, 74):
        at = torch.full((b,), t + 1, dtype=torch.int32, device=cuda)
        out = cfa.paged_attention(qt[:, :, t:t + 1], kp, vp, table, at, 0.125, **how)
        assert rel(out[:, :, 0], whole[:, :, t]) <= bar, t


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("cap", [None, 3.0], ids=["plain", "capped"])
def test_slopes_to_the_largest_float(cuda, d, causal, cap):
    """Slopes that are floats but not in units of log2 e, or not times a distance: a query's own key alone."""
    big = torch.finfo(torch.float32).max
    slopes = torch.tensor([big, 2.4e38, 1e38, 1e37])
    q, k, v, g = operands(2, 4, 2, 150, 300, d, seed=24)
    got = run(cuda, q, k, v, g, d ** -0.5, causal, cap=cap, slopes=slopes)
    ref, _ = formula(q, k, v, g, d ** -0.5, causal, cap=cap, slopes=slopes)
    check([got[0], got[3]], [ref[0], ref[3]])
    # (No gradient of the scores: P (dP - D) of a weight of 1, where dP and D are the same sum but for roundings.)
    assert all(float(x.abs().max()) <= 1e-5 for x in got[1:3])


@pytest.mark.parametrize("cap,scale,spread", [(1e30, 1e-9, 1e9), (1e30, 0.125, 1.0), (1e25, 1e-12, 1e12), (1e13, 1e-3, 1e3),
                                              (1e-13, 0.125, 1.0), (1e-30, 1e9, 1.0), (1e-30, 1e-9, 1.0)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_caps_to_the_ends(cuda, cap, scale, spread, d):
    """Caps whose quotient with the scale, and with the operands' units, leaves the range of floats; scores of 0
    among them. (x / cap is off by as much as x, so the scores' derivative by nothing that counts.)"""
    q, k, v, g = operands(1, 4, 2, 150, 180, d, seed=25, spread=spread)
    q[:, :, ::3] = 0.0
    for causal in (True, False):
        ref, top = formula(q, k, v, g, scale, causal, cap=cap)
        check(run(cuda, q, k, v, g, scale, causal, cap=cap), ref, top)
    slopes = torch.tensor([0.1, 0.0, 0.01, 1.5])
    ref, top = formula(q, k, v, g, scale, True, cap=cap, slopes=slopes)
    check(run(cuda, q, k, v, g, scale, True, cap=cap, slopes=slopes), ref, top)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_a_negative_scale_is_a_sign_of_the_queries(cuda, d, causal):
    """The same bits as of negated queries (by another path, in fp32, they would differ): scores that are hidden
    stay hidden whatever the scale's sign. (dK sums the queries themselves, whose signs a matrix instruction need not
    round alike.)"""
    ids = ids_of([[100, 130, 60], [300]], 300)
    q, k, v, g = operands(2, 4, 2, 200, 300, d, seed=26)
    for how in (dict(), dict(documents=ids), dict(cap=3.0), dict(slopes=torch.tensor([0.1, 0.0, 2.0, -0.01]))):
        got = run(cuda, q, k, v, g, -0.2, causal, **how)
        want = run(cuda, -q, k, v, g, 0.2, causal, **how)
        want[1] = -want[1]
        assert [torch.equal(got[i], want[i]) for i in (0, 1, 3)] == [True] * 3
        check(got, formula(q, k, v, g, -0.2, causal, **how)[0], 10.0)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("spread", [0.0, 1e-4, 1.0])
def test_rows_of_zeros(cuda, d, spread):
    """Padding of zeros behind a sample, and zero keys under small queries: where every score is 0 a score formed
    another way (less a slope of 0) has the same bits, those of fp32 would differ. Scale 0 likewise."""
    q, k, v, g = operands(2, 4, 2, 290, 300, d, seed=27)
    q[:, :, 150:] *= spread
    k[:, :, 160:] = 0.0
    for scale in (0.125, -0.125, 0.0):
        for causal in (True, False):
            got = run(cuda, q, k, v, g, scale, causal)
            check(got, formula(q, k, v, g, scale, causal)[0] if scale else
                  [torch.zeros_like(x, dtype=torch.float64) if i in (1, 2) else x
                   for i, x in enumerate(formula(q, k, v, g, 0.0, causal)[0])])
            if spread == 0.0 or scale == 0.0:
                other = run(cuda, q, k, v, g, scale, causal, slopes=torch.zeros(4))
                assert torch.equal(got[0][:, :, 192:], other[0][:, :, 192:])
                assert torch.equal(got[1][:, :, 192:], other[1][:, :, 192:])
                if causal:
                    assert torch.equal(got[3][:, :, 256:], other[3][:, :, 256:])
