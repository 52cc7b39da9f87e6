"""The paged cache on the GPU: paged_append and paged_attention against plain formulas in 64 bits, where
they can go wrong: lengths around the kernel's tiles and the pages' ends, empty sequences, ragged
counts, grouped heads in more than one block of rows, strided caches and operands, garbage behind the
last token, pages that the cache does not have, side streams and captured graphs.

Tolerances. A stored value is rounded once: half a step of its type. The attention's sums are fp32 of
N(0, 1) values: 2e-6 normwise, the bar of every fp32 attention test here; a 16-bit result is rounded
once more, at most eps / 2 of each value, so of the norm. (The weights' and fp32 queries' 16-bit terms
leave 2^-17 for 16-bit results, far below their rounding, and 2^-22 for fp32 ones.)"""
from __future__ import annotations

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def bar(dtype):
    return 2e-6 + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def rel(x, ref):
    """Normwise error of the worst row of head_dim values."""
    x, ref = x.double().cpu(), ref.double().cpu()
    n = ref.norm(dim=-1)
    return float(((x - ref).norm(dim=-1) / n.clamp_min(1e-30)).max()) if n.numel() else 0.0


class Cache:
    """A page pool of N(0, 1) values with NaN in every slot behind its sequence's length, and a table
    that deals the pages out in a shuffled order."""

    def __init__(self, dev, dtype, hk, page, d, lengths, room=0, seed=0, spare=2):
        gen = torch.Generator().manual_seed(seed)
        self.page, self.d, self.hk = page, d, hk
        per = [-(-(n + room) // page) for n in lengths]
        total = sum(per) + spare
        order = torch.randperm(total, generator=gen)
        width = max(1, max(per))
        self.table = torch.full((len(lengths), width), 10 ** 6, dtype=torch.int32)  # no such page
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.k = torch.full((total, hk, page, d), float("nan"))
        self.v = self.k.clone()
        for i, n in enumerate(lengths):
            for t0 in range(0, n, page):
                p, m = int(self.table[i, t0 // page]), min(page, n - t0)
                self.k[p, :, :m] = torch.randn(hk, m, d, generator=gen)
                self.v[p, :, :m] = torch.randn(hk, m, d, generator=gen)
        self.k, self.v = self.k.to(dtype).to(dev), self.v.to(dtype).to(dev)
        self.table = self.table.to(dev)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=dev)

    def dense(self, i, n):
        """Keys and values [hk, n, d] of sequence i, 64 bits, on the CPU."""
        pages = self.table[i, :-(-n // self.page)].long().cpu()
        return [x.cpu()[pages].transpose(0, 1).reshape(self.hk, -1, self.d)[:, :n].double()
                for x in (self.k, self.v)]


def attend(q, cache, lengths, scale):
    """The formula in 64 bits, one sequence at a time."""
    b, h, _, d = q.shape
    out = torch.zeros(b, h, 1, d, dtype=torch.float64)
    for i, n in enumerate(lengths):
        if n:
            k, v = cache.dense(i, n)
            x = torch.matmul(q[i, :, 0].double().cpu().view(cache.hk, -1, d),
                             k.transpose(1, 2).contiguous()) * scale
            out[i] = torch.matmul(torch.softmax(x, dim=-1), v).reshape(h, 1, d)
    return out


def q_of(dev, dtype, b, h, d, seed=1):
    return torch.randn(b, h, 1, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("types", PAIRS, ids="-".join)
def test_attention_types_and_head_dims(cuda, types, d):
    dt, ct = (TYPES[t] for t in types)
    lengths = [1, 15, 16, 17, 31, 32, 33, 0, 100, 129, 257, 511, 640]
    c = Cache(cuda, ct, 3, 32, d, lengths)
    q = q_of(cuda, dt, len(lengths), 6, d)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5)
    assert out.dtype == dt and out.shape == q.shape
    ref = attend(q, c, lengths, d ** -0.5)
    assert float(out[7].abs().max()) == 0.0
    assert rel(out, ref) <= bar(dt)
    assert torch.equal(out, cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5))


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("lengths", [[700, 1, 3000], [5000], [0, 0, 1025], [4097] * 9])
def test_attention_pages_and_splits(cuda, page, lengths):
    c = Cache(cuda, torch.float32, 2, page, 64, lengths, seed=3)
    q = q_of(cuda, torch.float32, len(lengths), 2, 64)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125)
    assert rel(out, attend(q, c, lengths, 0.125)) <= bar(torch.float32)


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16")], ids="-".join)
@pytest.mark.parametrize("h,hk", [(1, 1), (5, 1), (8, 2), (16, 1), (17, 1), (40, 1), (48, 2)])
def test_attention_grouped_heads(cuda, types, h, hk):
    dt, ct = (TYPES[t] for t in types)
    lengths = [70, 1300, 513]
    c = Cache(cuda, ct, hk, 32, 64, lengths, seed=4)
    q = q_of(cuda, dt, 3, h, 64)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125)
    assert rel(out, attend(q, c, lengths, 0.125)) <= bar(dt)


def test_attention_many_sequences(cuda):
    """More sequences than a workgroup has threads, empty ones among them."""
    lengths = [(37 * i) % 150 if i % 5 else 0 for i in range(700)] + [900]
    c = Cache(cuda, torch.float32, 1, 16, 32, lengths, seed=5)
    q = q_of(cuda, torch.float32, len(lengths), 1, 32)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.2)
    assert rel(out, attend(q, c, lengths, 0.2)) <= bar(torch.float32)


@pytest.mark.parametrize("types", PAIRS, ids="-".join)
def test_attention_large_and_sinking_scores(cuda, types):
    """Scores to +-100 in an order that moves the reference again and again, a negative scale, and one
    key of all the weight before many of little: those keep theirs."""
    dt, ct = (TYPES[t] for t in types)
    n = 1500
    c = Cache(cuda, ct, 1, 64, 64, [n], seed=6)
    q = q_of(cuda, dt, 1, 2, 64)
    for scale in (1.5, -1.5):
        out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, scale)
        # An exponent is off by half a step of its size, up to 2^7 (in log2 units), and the scores' sums
        # by as much again over d = 64 products; each weight by 2 x 2^7 x 2^-24 x ln 2 = 1.1e-5.
        assert rel(out, attend(q, c, [n], scale)) <= bar(dt) + 1.1e-5
    first = int(c.table[0, 0])
    u = torch.ones(64, device=cuda) / 8
    c.k.copy_(0.01 * torch.nan_to_num(c.k.float()))
    c.k[first, 0, 0] = (24.0 * u).to(ct)  # exp(24 - 0): e^-24 = 3.8e-11 each for the rest
    c.v[first, 0, 0] = 0.0
    q = (8 * u).to(dt).expand(1, 2, 1, 64).contiguous()
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 1.0 / 8)
    ref = attend(q, c, [n], 1.0 / 8)
    # (An f16 result of 1e-9 is below the least f16, 2^-24: each of 64 values is off by up to 2^-25.)
    least = 2.0 ** -25 * 8 / float(ref.norm(dim=-1).min()) if dt == torch.float16 else 0.0
    assert rel(out, ref) <= bar(dt) + 1.1e-5 + least


@pytest.mark.parametrize("types", PAIRS, ids="-".join)
@pytest.mark.parametrize("n", [70, 1500])
def test_attention_non_finite_values_that_are_seen(cuda, types, n):
    """Infinities among the values, a key that scores minus infinity, a NaN among the keys: what the formula
    gives, and nothing of them in other sequences, rows and columns. (The queries are halves of whole
    numbers, exact in every type, and not 0, so that the infinite key's score is one.)"""
    dt, ct = (TYPES[t] for t in types)
    c = Cache(cuda, ct, 1, 16, 64, [n] * 4, seed=18)
    q = ((torch.randint(1, 5, (4, 2, 1, 64), generator=torch.Generator().manual_seed(2)) / 2)
         .to(dt).to(cuda))

    def put(pages, i, t, e, value):
        pages[int(c.table[i, t // 16]), 0, t % 16, e] = value

    put(c.v, 0, 3, 5, float("inf")), put(c.v, 0, 40, 9, float("-inf"))
    put(c.k, 1, 7, 11, float("-inf"))
    put(c.k, 2, 9, 2, float("nan"))
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.05).double().cpu()
    ref = attend(q, c, [n] * 4, 0.05)
    assert torch.equal(out.isnan(), ref.isnan()) and bool(out[2].isnan().all())
    assert torch.equal(out.isinf(), ref.isinf()) and out[0, 0, 0, 5] > 0 > out[0, 0, 0, 9]
    fine = ref.isfinite()
    assert rel(out[fine][None], ref[fine][None]) <= bar(dt)


@pytest.mark.parametrize("types", PAIRS, ids="-".join)
@pytest.mark.parametrize("n", [70, 1500])
def test_attention_scores_of_minus_infinity(cuda, types, n):
    """Keys that score minus infinity have no weight, whole tiles and runs of them; an infinite value of one
    gives NaN (0 times infinity), and a sequence of nothing else is NaN, as the formula."""
    dt, ct = (TYPES[t] for t in types)
    c = Cache(cuda, ct, 1, 16, 64, [n] * 4, seed=19)
    q = ((torch.randint(1, 5, (4, 2, 1, 64), generator=torch.Generator().manual_seed(3)) / 2)
         .to(dt).to(cuda))
    for i, last in ((1, n * 2 // 3), (2, n), (3, n * 2 // 3)):
        for t in range(last):
            c.k[int(c.table[i, t // 16]), 0, t % 16, 9] = -float("inf")
    c.v[int(c.table[3, 2]), 0, 5, 4] = float("inf")
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.05).double().cpu()
    ref = attend(q, c, [n] * 4, 0.05)
    assert torch.equal(out.isnan(), ref.isnan()) and bool(ref[2].isnan().all())
    assert ref[3].isnan().sum() == 2 and bool(ref[1].isfinite().all())
    fine = ref.isfinite()
    assert rel(out[fine][None], ref[fine][None]) <= bar(dt)


def test_attention_strided_cache_and_queries(cuda):
    """Keys and values interleaved in one pool whose rows are padded and whose heads come after the
    slots; queries out of a wider buffer, misaligned ones copied."""
    lengths = [333, 77]
    c = Cache(cuda, torch.float32, 3, 16, 64, lengths, seed=7)
    pool = torch.full((c.k.shape[0], 16, 2, 3, 72), float("nan"), device=cuda)
    pool[:, :, 0, :, :64], pool[:, :, 1, :, :64] = c.k.transpose(1, 2), c.v.transpose(1, 2)
    kp, vp = (pool[:, :, i, :, :64].transpose(1, 2) for i in range(2))
    table = torch.full((2, 40), -1, dtype=torch.int32, device=cuda)
    table[:, :c.table.shape[1]] = c.table
    wide = torch.randn(2, 3, 1, 3 * 64, device=cuda)
    for q in (wide[..., 64:128], wide[..., 1:65]):
        out = cfa.paged_attention(q, kp, vp, table[:, :c.table.shape[1]], c.lengths, 0.125)
        assert rel(out, attend(q, c, lengths, 0.125)) <= bar(torch.float32)


@pytest.mark.parametrize("capacity_pages", [4, 200])
def test_attention_bad_pages_and_lengths(cuda, capacity_pages):
    """Pages the cache does not have, and lengths the table does not hold: NaN in those sequences alone,
    on both sides of the choice between one workgroup per head and shared ones."""
    lengths = [60, 60, 60, 60, 60]
    c = Cache(cuda, torch.float32, 2, 16, 64, lengths, seed=8)
    table = torch.zeros(5, capacity_pages, dtype=torch.int32, device=cuda)
    table[:, :4] = c.table[:, :4]
    table[1, 2], table[2, 3] = c.k.shape[0], -1
    c.lengths[3], c.lengths[4] = -1, capacity_pages * 16 + 1
    q = q_of(cuda, torch.float32, 5, 4, 64)
    out = cfa.paged_attention(q, c.k, c.v, table, c.lengths, 0.125)
    assert rel(out[:1], attend(q[:1], c, [60], 0.125)) <= bar(torch.float32)
    assert bool(out[1:].isnan().all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("types", PAIRS, ids="-".join)
def test_append(cuda, types, interleaved):
    """Ragged new tokens behind what the caches hold: the written slots against the formula, every other
    slot untouched, q turned in all its rows."""
    dt, ct = (TYPES[t] for t in types)
    held, counts, s, h, hk, d, dim = [0, 5, 31, 100], [7, 0, 40, 33], 40, 4, 2, 64, 32
    c = Cache(cuda, ct, hk, 16, d, held, room=s, seed=9)
    gen = torch.Generator().manual_seed(10)
    q, k, v = (torch.randn(4, s, n, d, generator=gen).to(dt).to(cuda).transpose(1, 2) for n in (h, hk, hk))
    f = cfa.rotary_frequencies(dim, device=cuda)
    before = c.k.clone(), c.v.clone()
    qr = cfa.paged_append(k, v, c.k, c.v, c.table, c.lengths,
                          counts=torch.tensor(counts, dtype=torch.int32, device=cuda), q=q,
                          frequencies=f, interleaved=interleaved)
    pos = (c.lengths.long().cpu()[:, None] + torch.arange(s))[:, None, :, None]
    a = pos.double() * f.cpu()

    def turn(x):
        x = x.double().cpu()
        y, m = x.clone(), dim // 2
        i, j = (slice(0, dim, 2), slice(1, dim, 2)) if interleaved else (slice(0, m), slice(m, dim))
        y[..., i] = x[..., i] * a.cos() - x[..., j] * a.sin()
        y[..., j] = x[..., j] * a.cos() + x[..., i] * a.sin()
        return y

    def near(x, ref, size):
        # Four 32-bit roundings of a pair's terms, and half a step of the stored type.
        eps = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
        tiny = 0.0 if x.dtype != torch.float16 else 2.0 ** -25  # half a step of subnormal f16
        assert bool(((x.double().cpu() - ref).abs() <= 4 * 2.0 ** -24 * size + eps * ref.abs() * 1.0001
                     + tiny).all())

    near(qr, turn(q), 2 * q.double().cpu().abs().amax(-1, keepdim=True))
    kt, untouched = turn(k), torch.ones(c.k.shape[0], 16, dtype=torch.bool)
    for i, (have, new) in enumerate(zip(held, counts)):
        for t in range(new):
            p, slot = int(c.table[i, (have + t) // 16]), (have + t) % 16
            untouched[p, slot] = False
            near(c.k[p, :, slot], kt[i, :, t], 2 * k[i, :, t].double().cpu().abs().amax(-1, keepdim=True))
            assert torch.equal(c.v[p, :, slot], v[i, :, t].to(ct))
    for x, y in zip((c.k, c.v), before):
        x, y = (z.cpu().transpose(1, 2)[untouched] for z in (x, y))
        assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))


def test_append_without_rotation_queries_or_pages(cuda):
    """Plain copies; tokens whose page is missing, out of the cache, or past the table are dropped, and so
    is a sequence of negative length."""
    c = Cache(cuda, torch.bfloat16, 1, 16, 32, [0, 0, 0, 0], room=32, seed=11)
    c.k.zero_(), c.v.zero_()
    k, v = (torch.randn(4, 1, 40, 32, device=cuda) for _ in range(2))
    table = c.table.clone()
    table[1, 0], table[2, 1] = -1, c.k.shape[0]
    c.lengths[3] = -5
    assert cfa.paged_append(k, v, c.k, c.v, table, c.lengths) is None
    for x, pages in ((k, c.k), (v, c.v)):
        want = torch.zeros_like(pages)
        x = x.to(torch.bfloat16)[:, 0]
        want[int(table[0, 0]), 0], want[int(table[0, 1]), 0] = x[0, :16], x[0, 16:32]
        want[int(table[1, 1]), 0], want[int(table[2, 0]), 0] = x[1, 16:32], x[2, :16]
        assert torch.equal(pages, want)


def test_append_odd_layouts(cuda):
    """Operands that only single values can be read of: an odd offset, and a rotated part of 2 x 3."""
    c = Cache(cuda, torch.float32, 2, 16, 32, [3, 0], room=4, seed=12)
    buf = torch.randn(2 * 2 * 4 * 33 + 1, device=cuda)
    k = buf[1:].view(2, 2, 4, 33)[..., :32]
    v = torch.randn(2, 2, 4, 32, device=cuda)
    f = cfa.rotary_frequencies(6, device=cuda)
    for interleaved in (False, True):
        a, b = (Cache(cuda, torch.float32, 2, 16, 32, [3, 0], room=4, seed=12) for _ in range(2))
        cfa.paged_append(k, v, a.k, a.v, a.table, a.lengths, frequencies=f, interleaved=interleaved)
        cfa.paged_append(k.contiguous(), v, b.k, b.v, b.table, b.lengths, frequencies=f,
                         interleaved=interleaved)
        assert torch.equal(a.k.nan_to_num(9.0), b.k.nan_to_num(9.0))
        assert torch.equal(a.v.nan_to_num(9.0), b.v.nan_to_num(9.0))


def test_decoding_run_equals_prompt_attention(cuda):
    """A prompt through fused_rotary and fused_attention, and the same tokens one by one through
    paged_append and paged_attention (the first half appended at once): the same rows."""
    b, h, s, d = 2, 3, 40, 64
    gen = torch.Generator(device=cuda).manual_seed(13)
    q, k, v = (torch.randn(b, h, s, d, device=cuda, generator=gen) for _ in range(3))
    f = cfa.rotary_frequencies(d, device=cuda)
    qr, kr = cfa.fused_rotary(q, k, torch.arange(s, device=cuda), f)
    want = cfa.fused_attention(qr, kr, v, 0.125, True)
    c = Cache(cuda, torch.float32, h, 16, d, [0] * b, room=s, seed=14)
    lengths = torch.zeros(b, dtype=torch.int32, device=cuda)
    cfa.paged_append(k[:, :, :20], v[:, :, :20], c.k, c.v, c.table, lengths, frequencies=f)
    lengths += 20
    for t in range(20, s):
        at = slice(t, t + 1)
        qt = cfa.paged_append(k[:, :, at], v[:, :, at], c.k, c.v, c.table, lengths, q=q[:, :, at],
                              frequencies=f)
        lengths += 1
        out = cfa.paged_attention(qt, c.k, c.v, c.table, lengths, 0.125)
        assert rel(out, want[:, :, at]) <= 2 * bar(torch.float32)


def test_decoding_step_captured(cuda):
    """A decoding step in a graph, replayed with other tokens, lengths and tables in the same buffers,
    eager work between: each replay equals the eager calls bit for bit."""
    b, h, hk, d = 3, 4, 2, 64
    c = Cache(cuda, torch.bfloat16, hk, 16, d, [900, 40, 0], room=32, seed=15)
    c.k.nan_to_num_(0.5), c.v.nan_to_num_(0.5)
    f = cfa.rotary_frequencies(d, device=cuda)
    q, k, v = (torch.randn(b, n, 1, d, device=cuda).bfloat16() for n in (h, hk, hk))
    lengths = c.lengths.clone()

    def step(kp, vp):
        qt = cfa.paged_append(k, v, kp, vp, c.table, lengths, q=q, frequencies=f)
        lengths.add_(1)
        return cfa.paged_attention(qt, kp, vp, c.table, lengths, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kp, vp = c.k.clone(), c.v.clone()
    with torch.cuda.stream(side):
        step(kp.clone(), vp.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(kp, vp)
    ek, ev, el = c.k.clone(), c.v.clone(), c.lengths.clone()
    kp.copy_(c.k), vp.copy_(c.v), lengths.copy_(c.lengths)
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        graph.replay()
        out = got.clone()
        qt = cfa.paged_append(k, v, ek, ev, c.table, el, q=q, frequencies=f)
        el += 1
        want = cfa.paged_attention(qt, ek, ev, c.table, el, 0.125)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    assert torch.equal(kp, ek) and torch.equal(vp, ev) and torch.equal(lengths, el)


def test_attention_side_streams(cuda):
    """Two calls in flight on two streams, each with its own workspace."""
    c = Cache(cuda, torch.float32, 2, 16, 64, [5000, 700], seed=16)
    qs = [q_of(cuda, torch.float32, 2, 2, 64, seed=i) for i in range(2)]
    want = [cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cfa.paged_attention(qs[i], c.k, c.v, c.table, c.lengths, 0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_append_refuses_one_cache_for_both(cuda):
    c = Cache(cuda, torch.float32, 2, 16, 64, [3])
    x = torch.zeros(1, 2, 1, 64, device=cuda)
    with pytest.raises(cfa.FusedAttentionError, match="same memory"):
        cfa.paged_append(x, x, c.k, c.k, c.table, c.lengths)


def test_append_refuses_broadcast_pages(cuda):
    c = Cache(cuda, torch.float32, 1, 16, 32, [5], room=2, seed=17)
    k = torch.randn(1, 2, 2, 32, device=cuda)
    with pytest.raises(cfa.FusedAttentionError, match="broadcast"):
        cfa.paged_append(k, k, c.k.expand(-1, 2, -1, -1), c.v.expand(-1, 2, -1, -1), c.table, c.lengths)


def test_far_pages(cuda):
    """A pool of more than 2^31 values, its last pages in use: as a small pool, bit for bit."""
    far = torch.empty(2, 70000, 8, 64, 64, dtype=torch.bfloat16, device=cuda)
    near = torch.zeros(2, 3, 8, 64, 64, dtype=torch.bfloat16, device=cuda)
    far[:, -3:] = 0
    k, v = (torch.randn(1, 8, 130, 64, device=cuda).bfloat16() for _ in range(2))
    q = q_of(cuda, torch.bfloat16, 1, 16, 64, seed=19)
    zero, n = (torch.tensor([i], dtype=torch.int32, device=cuda) for i in (0, 130))
    out = []
    for pool, first in ((far, 69997), (near, 0)):
        table = torch.tensor([[first + 2, first, first + 1]], dtype=torch.int32, device=cuda)
        cfa.paged_append(k, v, pool[0], pool[1], table, zero)
        out.append(cfa.paged_attention(q, pool[0], pool[1], table, n, 0.125))
    assert torch.equal(far[:, -3:], near) and torch.equal(*out)
    assert bool(out[0].isfinite().all()) and float(out[0].abs().max()) > 0


def test_append_side_stream(cuda):
    """On another stream than the default one, ordered by events: as on the default."""
    a, b = (Cache(cuda, torch.float32, 2, 16, 64, [9, 0], room=300, seed=20) for _ in range(2))
    k, v, q = (torch.randn(2, n, 300, 64, device=cuda) for n in (2, 2, 4))
    f = cfa.rotary_frequencies(64, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = cfa.paged_append(k, v, a.k, a.v, a.table, a.lengths, q=q, frequencies=f)
    torch.cuda.current_stream().wait_stream(side)
    y = cfa.paged_append(k, v, b.k, b.v, b.table, b.lengths, q=q, frequencies=f)
    assert torch.equal(x, y)
    assert all(torch.equal(s.nan_to_num(9.0), t.nan_to_num(9.0)) for s, t in ((a.k, b.k), (a.v, b.v)))


@pytest.mark.parametrize("width", [1, 100])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_16_bit_results_are_rounded_once(cuda, dtype, width):
    """A 16-bit result is off by half a step of its own and an error of fp32 sums, no more: as far from the
    exact value as its rounding, but where that lies within 2^-19 of the values' size of a tie. Tables as
    wide as the sequences, and far wider.

    Scores are exact (halves times halves, a scale of 2^-8, so at most 1/2 and 0.72 in log2 units). In
    units of 2^-24: log2 e and the exponent are off by 0.72 each and their difference by 1.44, by ln 2 of a
    weight: 2; the exponential by 2; so 8 for the weights above and below the line, 16 for the sum of 4 keys
    on the matrix instructions, 5 for that of the weights, 3 for the quotient: 32, 2^-19."""
    b, h, d, n, dt = 128, 16, 128, 4, TYPES[dtype]
    gen = torch.Generator().manual_seed(22)
    halves = lambda *shape: (torch.randint(0, 4, shape, generator=gen) - 1.5).sign() * (
        torch.randint(1, 3, shape, generator=gen) / 2)
    q, k = halves(b, h, 1, d), halves(b, h, n, d)
    v = torch.randn(b, h, n, d, generator=gen).to(dt)
    kp, vp = (torch.full((b, h, 16, d), float("nan"), dtype=dt) for _ in range(2))
    kp[:, :, :n], vp[:, :, :n] = k.to(dt), v
    table = torch.full((b, width), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(b)
    out = cfa.paged_attention(q.to(dt).to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda),
                              torch.full((b,), n, dtype=torch.int32, device=cuda), 2.0 ** -8)
    p = torch.softmax(torch.matmul(q.double(), k.double().transpose(2, 3).contiguous()) * 2.0 ** -8, -1)
    ref, size = torch.matmul(p, v.double()), torch.matmul(p, v.double().abs())
    room = 2.0 ** -19 * size
    # Half a step at the value (the least normal f16 is 2^-14).
    least = 2.0 ** -14 if dt == torch.float16 else 2.0 ** -126
    half = torch.exp2(torch.floor(torch.log2((ref.abs() + room).clamp_min(least)))) * (torch.finfo(dt).eps / 2)
    over = (out.double().cpu() - ref).abs() - half - room
    assert int((over > 0).sum()) == 0, (int((over > 0).sum()), float((over / size).max()))


@pytest.mark.parametrize("types", PAIRS, ids="-".join)
def test_append_overlapping_operands(cuda, types):
    """New keys, values and queries whose rows overlap (windows of a longer row): as of contiguous copies,
    bit for bit."""
    dt, ct = (TYPES[t] for t in types)
    buf = torch.randn(4096, generator=torch.Generator().manual_seed(23)).to(dt).to(cuda)
    k, v, q = (buf.as_strided((2, n, 20, 64), (700, 100, 1, 1), i) for i, n in enumerate((2, 2, 4)))
    f = cfa.rotary_frequencies(64, device=cuda)
    a, b = (Cache(cuda, ct, 2, 16, 64, [5, 30], room=20, seed=24) for _ in range(2))
    x = cfa.paged_append(k, v, a.k, a.v, a.table, a.lengths, q=q, frequencies=f)
    y = cfa.paged_append(k.contiguous(), v.contiguous(), b.k, b.v, b.table, b.lengths, q=q.contiguous(),
                         frequencies=f)
    assert torch.equal(x, y)
    assert all(torch.equal(s.nan_to_num(9.0), t.nan_to_num(9.0)) for s, t in ((a.k, b.k), (a.v, b.v)))


def test_append_counts_as_a_write_of_the_pages(cuda):
    """The pages' versions move with an append, and nothing else's: a graph that saved pages before it
    refuses its backward, which would run on other values. Pages without versions (inference mode) are
    written all the same."""
    c = Cache(cuda, torch.float32, 2, 16, 64, [3, 0], room=2, seed=21)
    k, v, q = (torch.randn(2, n, 2, 64, device=cuda) for n in (2, 2, 4))
    f = cfa.rotary_frequencies(64, device=cuda)
    w = torch.ones((), device=cuda, requires_grad=True)
    losses = [(w * pages[:1]).sum() for pages in (c.k, c.v)]
    others = (k, v, q, f, c.table, c.lengths)
    before = [t._version for t in (c.k, c.v, *others)]
    cfa.paged_append(k, v, c.k, c.v, c.table, c.lengths, q=q, frequencies=f)
    after = [t._version for t in (c.k, c.v, *others)]
    assert after == [before[0] + 1, before[1] + 1, *before[2:]]
    for loss in losses:
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        kp, vp = c.k.nan_to_num(0.0), c.v.nan_to_num(0.0)
        cfa.paged_append(2.0 * k, v, kp, vp, c.table, c.lengths)
        assert torch.equal(kp[int(c.table[1, 0]), :, :2], 2.0 * k[1])
