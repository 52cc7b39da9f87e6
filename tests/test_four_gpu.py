"""The paged cache in 4 bits, tokens back out of a cache, and one token's attention with capped and biased
scores, on the GPU against plain formulas in 64 bits: values on and next to the borders between codes,
groups with values that are not finite, partly rotated heads, unaligned operands, missing pages, slots that
must stay as they were, lengths around the tiles and pages, prompts against single tokens, captured steps.

Tolerances. Codes, and values read back, are exact. The attention's are those of the other caches' tests
(2e-6 normwise in fp32, half a step of a 16-bit result more); a capped or biased score y carries, next to
the plain score's error, that of x / cap, tanh (1.3 x 2^-24), the product with cap and the difference: 5 x
2^-24 of |y|, which is a weight's relative error, over the keys that weigh anything."""
from __future__ import annotations

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def encode(x):
    """Bytes of x [..., d] (64 bits, CPU): for each value the nearest of all fifteen, by distance."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    fine = top.isfinite()
    e = torch.full(top.shape, -127.0, dtype=torch.float64)
    for k in range(-127, 130):
        e = torch.where(top > 7 * 2.0 ** k, torch.tensor(float(k + 1), dtype=torch.float64), e)
    u = torch.where(fine[..., None], (g / torch.exp2(e)[..., None]).abs(), torch.zeros((), dtype=torch.float64))
    far = (u[..., None] - LEVELS).abs()
    best = far.amin(-1, keepdim=True)
    # (Of two at the same distance the even one.)
    code = torch.where(far == best, torch.tensor([0, 9, 2, 11, 4, 13, 6, 15]), 99).amin(-1) % 8
    code = torch.where((g < 0) & (code > 0), code + 8, code).flatten(-2).byte()
    scale = torch.where(fine, e + 127, torch.tensor(255.0, dtype=torch.float64)).byte()
    pad = torch.zeros(*x.shape[:-1], -scale.shape[-1] % 4, dtype=torch.uint8)
    return torch.cat((code[..., 0::2] + 16 * code[..., 1::2], scale, pad), -1)


def decode(rows, d):
    """The values of bytes, in 64 bits on the CPU."""
    rows = rows.cpu()
    codes = torch.stack((rows[..., :d // 2] & 15, rows[..., :d // 2] >> 4), -1).flatten(-2).long()
    scale = rows[..., d // 2:d // 2 + d // 32].double()
    scale = torch.where(scale == 255, torch.tensor(float("nan"), dtype=torch.float64), torch.exp2(scale - 127))
    return torch.cat((LEVELS, -LEVELS))[codes] * scale.repeat_interleave(32, -1)


def turned(x, positions, f, interleaved, magnitude=1.0):
    """x [h, s, d] in 64 bits, turned at `positions`."""
    n = f.numel()
    a = positions.double()[:, None] * f.cpu()
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
    x = x.double().cpu().clone()
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    p, q = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo], x[..., hi] = p * c - q * s, q * c + p * s
    return x


class Four:
    """A 4-bit cache of random codes: bytes of 0xAA in every slot behind its sequence's length."""

    def __init__(self, dev, hk, page, d, lengths, room=0, seed=0, spare=1):
        gen = torch.Generator().manual_seed(seed)
        self.page, self.d, self.hk = page, d, hk
        per = [-(-(n + room) // page) for n in lengths]
        order = torch.randperm(sum(per) + spare, generator=gen)
        self.table = torch.full((len(lengths), max(1, max(per))), 10 ** 6, dtype=torch.int32)
        pools = [torch.full((sum(per) + spare, hk, page, cfa.fp4_row_bytes(d)), 0xAA, dtype=torch.uint8)
                 for _ in range(2)]
        self.spare, at = int(order[-1]), 0
        for i, (n, m) in enumerate(zip(lengths, per)):
            self.table[i, :m] = order[at:at + m].to(torch.int32)
            at += m
            for pool in pools:
                rows = encode(torch.randn(hk, n, d, generator=gen))
                for t in range(0, n, page):
                    pool[int(self.table[i, t // page]), :, :min(page, n - t)] = rows[:, t:t + page]
        self.k, self.v = (pool.to(dev) for pool in pools)
        self.table, self.lengths = self.table.to(dev), ints(lengths, dev)

    def dense(self, i, n):
        pages = self.table[i, :-(-n // self.page)].long().cpu()
        return [decode(x.cpu()[pages].transpose(0, 1).flatten(1, 2)[:, :n], self.d) for x in (self.k, self.v)]


def scores_of(q, k, scale, cap, slopes):
    """Scores [h, n] in 64 bits of one token's q [h, d] over k [hk, n, d]."""
    hk, n, d = k.shape
    y = torch.matmul(q.double().cpu().reshape(hk, -1, d), k.transpose(1, 2).contiguous()).flatten(0, 1) * scale
    if cap:
        y = cap * torch.tanh(y / cap)
    if slopes is not None:
        y = y - slopes.double().cpu()[:, None] * torch.arange(n - 1, -1, -1, dtype=torch.float64)
    return y


def attended(q, cache, lengths, scale, cap=None, slopes=None):
    """The formula in 64 bits, and the largest |y| of a key that weighs 1e-3 of its row's heaviest."""
    out, top = torch.zeros(q.shape, dtype=torch.float64), 0.0
    for i, n in enumerate(lengths):
        if n:
            k, v = cache.dense(i, n)
            y = scores_of(q[i, :, 0], k, scale, cap, slopes)
            p = torch.softmax(y, -1)
            if cap or slopes is not None:
                top = max(top, float(y[p > 1e-3 * p.amax(-1, keepdim=True)].abs().max()))
            out[i, :, 0] = torch.matmul(p.reshape(cache.hk, -1, n), v).flatten(0, 1)
    return out, top


def rel(x, ref):
    x, ref = x.double().cpu(), ref.double().cpu()
    return float(((x - ref).norm(dim=-1) / ref.norm(dim=-1).clamp_min(1e-30)).max()) if ref.numel() else 0.0


def bar(dtype, top=0.0):
    return 2e-6 + 5 * 2.0 ** -24 * top + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def q_of(dev, dtype, b, h, d, seed=1, spread=1.0):
    return (torch.randn(b, h, 1, d, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).to(dev)


# --- Appends ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,dim", [(32, 32), (32, 8), (64, 64), (64, 0), (64, 36), (128, 128), (128, 64)])
def test_append_codes(cuda, d, dim, dtype, interleaved):
    """Every byte of the pages, with new tokens into used caches of other lengths, past counts and missing
    pages, at positions past a hundred thousand too; and the turned queries, as fused_rotary's."""
    dt, held, counts = TYPES[dtype], [0, 5, 31, 100000], [40, 17, 0, 33]
    gen = torch.Generator().manual_seed(d + dim)
    c = Four(cuda, 2, 16, d, [0, 5, 31, 5], room=45, seed=2)
    c.table[3] = 10 ** 6
    wide = torch.full((4, 100040 // 16 + 1), -7, dtype=torch.int32, device=cuda)
    wide[:, :c.table.shape[1]] = c.table
    wide[3, 100000 // 16:100000 // 16 + 2] = ints([c.spare, 10 ** 7], cuda)  # (the spare page, and none)
    k, v, q = (torch.randn(4, n, 40, d, generator=gen).to(dt).to(cuda) for n in (2, 2, 6))
    f = cfa.rotary_frequencies(dim, device=cuda) if dim else None
    want = [c.k.cpu().clone(), c.v.cpu().clone()]
    for i, (n, m) in enumerate(zip(held, counts)):
        at = torch.arange(n, n + m)
        for pool, x, turn in ((want[0], k, dim > 0), (want[1], v, False)):
            x = x[i, :, :m]
            rows = encode(turned(x, at, f, interleaved, 1.25) if turn else x.cpu())
            for j, t in enumerate(at.tolist()):
                page = int(wide[i, t // 16])
                if 0 <= page < pool.shape[0]:
                    pool[page, :, t % 16] = rows[:, j]
    out = cfa.paged_append(k, v, c.k, c.v, wide, ints(held, cuda), counts=ints(counts, cuda), q=q,
                           frequencies=f, interleaved=interleaved, magnitude=1.25)
    assert torch.equal(c.k.cpu(), want[0]) and torch.equal(c.v.cpu(), want[1])
    if dim:
        pos = ints(held, cuda)[:, None] + torch.arange(40, device=cuda)
        assert torch.equal(out, cfa.fused_rotary(q, q, pos, f, interleaved, 1.25)[0])
    else:
        assert torch.equal(out, q)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_borders_and_extremes(cuda, dtype):
    """Values on the borders and a step of the type to either side, at scales to the type's ends; groups of
    zeros of both signs, of subnormals, with an infinity or NaN in one place, with one large value."""
    dt = TYPES[dtype]
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    ones = torch.cat([border, -border, LEVELS.float(), -LEVELS.float()])
    rows = []
    for e in (-126, -125, -30, -14, -3, 0, 5, 12, 30, 123, 124):
        x = (ones * 2.0 ** e).to(dt)
        one = x.view(torch.int32 if dt == torch.float32 else torch.int16)
        rows += [x, (one + 1).view(dt), torch.where(one.to(torch.int64) % 2 ** 15 > 0, one - 1, one).view(dt)]
    tiny = torch.full((32,), torch.finfo(dt).smallest_normal / 8, dtype=dt)
    rows += [torch.zeros(32, dtype=dt), -torch.zeros(32, dtype=dt), tiny, -tiny,
             torch.full((32,), torch.finfo(dt).max, dtype=dt)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = torch.randn(32).to(dt)
        x[7] = bad
        rows.append(x)
    x = torch.randn(32).to(dt)
    x[31] = 1000.0
    rows.append(x)
    x = torch.stack(rows)
    want = encode(x)
    n = len(rows)
    kp, vp = (torch.full((n // 16 + 1, 1, 16, 20), 7, dtype=torch.uint8, device=cuda) for _ in range(2))
    table = torch.arange(n // 16 + 1, dtype=torch.int32, device=cuda)[None]
    k = x.to(cuda)[None, None]
    cfa.paged_append(k, -k, kp, vp, table, ints([0], cuda))
    got = kp.flatten(0, 2)[:n].cpu()
    assert torch.equal(got, want), [(i, rows[i], got[i], want[i]) for i in range(n) if not torch.equal(got[i], want[i])][:3]
    assert torch.equal(vp.flatten(0, 2)[:n].cpu(), encode(-x))
    assert bool((kp.flatten(0, 2)[n:] == 7).all())
    for to in (torch.float32, torch.bfloat16):
        back, _ = cfa.paged_read(kp, vp, table, ints([n], cuda), n, dtype=to)
        ref = decode(want, 32).to(torch.float32).to(to)
        assert torch.equal(back[0, 0].cpu().nan_to_num(9e9), ref.nan_to_num(9e9))
        assert torch.equal(back[0, 0].cpu().isnan(), ref.isnan())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["odd base", "odd strides", "head views", "overlapping"])
def test_append_operands(cuda, dtype, kind):
    """Operands of other strides and alignments: the bytes of contiguous copies."""
    dt, gen = TYPES[dtype], torch.Generator().manual_seed(5)
    buf = torch.randn(60000, generator=gen).to(dt).to(cuda)
    st = {"odd base": (9000, 4000, 64, 1), "odd strides": (9001, 4001, 67, 1), "head views": (9600, 64, 192, 1),
          "overlapping": (700, 100, 1, 1)}[kind]
    k, v, q = (buf.as_strided((2, n, 50, 64), st, i) for i, n in ((1, 2), (3, 2), (6, 4)))
    f = cfa.rotary_frequencies(64, device=cuda)
    a, b = (Four(cuda, 2, 16, 64, [5, 30], room=50, seed=6) for _ in range(2))
    x = cfa.paged_append(k, v, a.k, a.v, a.table, a.lengths, q=q, frequencies=f)
    y = cfa.paged_append(k.contiguous(), v.contiguous(), b.k, b.v, b.table, b.lengths, q=q.contiguous(),
                         frequencies=f)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(x, y)


def test_append_prompt_or_single_tokens(cuda):
    """The same bytes in one call and token by token, on another stream, and into strided pages."""
    gen = torch.Generator().manual_seed(7)
    k, v = (torch.randn(2, 3, 37, 128, generator=gen).bfloat16().to(cuda) for _ in range(2))
    f = cfa.rotary_frequencies(128, device=cuda)
    a, b, c = (Four(cuda, 3, 16, 128, [0, 20], room=37, seed=8) for _ in range(3))
    cfa.paged_append(k, v, a.k, a.v, a.table, a.lengths, frequencies=f)
    lengths, side = b.lengths.clone(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(37):
            cfa.paged_append(k[:, :, i:i + 1], v[:, :, i:i + 1], b.k, b.v, b.table, lengths, frequencies=f)
            lengths += 1
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    pool = torch.zeros(a.k.shape[0], 16, 2, 3, 80, dtype=torch.uint8, device=cuda)
    kp, vp = (pool[:, :, i, :, 4:72].transpose(1, 2) for i in range(2))
    kp.copy_(c.k), vp.copy_(c.v)
    cfa.paged_append(k, v, kp, vp, c.table, c.lengths, frequencies=f)
    assert torch.equal(kp, a.k) and torch.equal(vp, a.v)
    assert int(pool[..., :4].max()) == 0 and int(pool[..., 72:].max()) == 0
    q = q_of(cuda, torch.float32, 2, 6, 128)
    lengths = ints([37, 57], cuda)
    assert torch.equal(cfa.paged_attention(q, kp, vp, c.table, lengths, 0.1),
                       cfa.paged_attention(q, a.k, a.v, a.table, lengths, 0.1))


# --- Attention over 4 bits --------------------------------------------------------------------------


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mods", [(None, False), (4.0, False), (30.0, True)], ids=["plain", "capped", "both"])
def test_attention_lengths(cuda, dtype, d, mods):
    dt, (cap, biased) = TYPES[dtype], mods
    lengths = [1, 15, 16, 17, 31, 32, 33, 0, 100, 129, 257, 511, 640]
    c = Four(cuda, 3, 32, d, lengths)
    q = q_of(cuda, dt, len(lengths), 6, d, spread=3.0)
    slopes = torch.tensor([0.5, 0.25, 0.0, 2.0, -0.01, 1e-3], device=cuda) if biased else None
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5, cap=cap, slopes=slopes)
    ref, top = attended(q, c, lengths, d ** -0.5, cap, slopes)
    assert out.dtype == dt and float(out[7].abs().max()) == 0.0
    assert rel(out, ref) <= bar(dt, max(top, 10.0))
    assert torch.equal(out, cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5, cap=cap, slopes=slopes))


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("lengths", [[700, 1, 3001], [5000], [0, 0, 1025], [4097] * 5])
def test_attention_pages_and_splits(cuda, page, lengths):
    c = Four(cuda, 2, page, 64, lengths, seed=3)
    q = q_of(cuda, torch.float32, len(lengths), 8, 64)
    slopes = torch.exp2(-torch.arange(8.0, device=cuda))
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, slopes=slopes)
    ref, top = attended(q, c, lengths, 0.125, None, slopes)
    assert rel(out, ref) <= bar(torch.float32, top)


@pytest.mark.parametrize("h,hk", [(1, 1), (17, 1), (40, 1), (48, 2)])
def test_attention_grouped_heads(cuda, h, hk):
    """More rows than a block has: each head's own slope."""
    lengths = [70, 1300, 513]
    c = Four(cuda, hk, 32, 64, lengths, seed=4)
    q = q_of(cuda, torch.bfloat16, 3, h, 64)
    slopes = torch.linspace(0.001, 1.0, h, device=cuda)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, cap=20.0, slopes=slopes)
    ref, top = attended(q, c, lengths, 0.125, 20.0, slopes)
    assert rel(out, ref) <= bar(torch.bfloat16, top)


@pytest.mark.parametrize("b,hk,most", [(32, 6, 1280), (32, 6, 1312), (64, 8, 2048), (64, 8, 2080)])
def test_attention_batches(cuda, b, hk, most):
    """Batches that a workgroup per key head takes, and the next capacity, that it does not."""
    gen = torch.Generator().manual_seed(most)
    lengths = [most, 0, 1, most - 1] + torch.randint(1, most, (b - 4,), generator=gen).tolist()
    c = Four(cuda, hk, 32, 32, lengths, seed=10)
    q = q_of(cuda, torch.float32, b, hk, 32)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.2)
    ref, top = attended(q, c, lengths, 0.2)
    assert rel(out, ref) <= bar(torch.float32, max(top, 10.0))


def test_attention_bad_sequences_and_groups(cuda):
    """A length or a page that the cache does not have: NaN there, the neighbours as they are. A group of
    NaN: seen as a value in its own 32 head_dims, as a key everywhere; behind the last token not at all."""
    c = Four(cuda, 2, 16, 64, [50, 50, 50, 50, 50], seed=9)
    q = q_of(cuda, torch.float32, 5, 4, 64)
    good = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, cap=9.0)
    ref, top = attended(q, c, [50] * 5, 0.125, 9.0)
    assert rel(good, ref) <= bar(torch.float32, top)
    lengths = c.lengths.clone()
    lengths[1] = -1
    table = c.table.clone()
    table[2, 2] = 10 ** 6
    k, v = c.k.clone(), c.v.clone()
    k[int(table[3, 1]), 1, 3, 33], v[int(table[4, 0]), 0, 5, 32] = 255, 255
    k[int(table[0, 3]), :, 2:, 32:34] = v[int(table[0, 3]), :, 2:, 32:34] = 255  # (tokens 50 on)
    out = cfa.paged_attention(q, k, v, table, lengths, 0.125, cap=9.0)
    assert torch.equal(out[0], good[0])
    assert bool(out[1].isnan().all()) and bool(out[2].isnan().all())
    assert torch.equal(out[3, :2], good[3, :2]) and bool(out[3, 2:].isnan().all())
    assert bool(out[4, :2, :, :32].isnan().all()) and torch.equal(out[4, :2, :, 32:], good[4, :2, :, 32:])
    assert torch.equal(out[4, 2:], good[4, 2:])


def test_attention_f16_queries_are_held_whole(cuda):
    """f16 queries of 11 significant bits, whose low bits decide: keys of one value, +-1."""
    d, n = 64, 2
    rows = encode(torch.cat([torch.ones(1, d), torch.ones(1, d) * torch.tensor([1.0, -1.0]).repeat(d // 2)]))
    kp = torch.zeros(1, 1, 16, 36, dtype=torch.uint8)
    kp[0, 0, :2] = rows
    vp = kp.clone()
    kp, vp = kp.to(cuda), vp.to(cuda)
    q = (1.0 + torch.arange(d) * 2.0 ** -10).to(torch.float16).view(1, 1, 1, d).to(cuda)
    out = cfa.paged_attention(q, kp, vp, ints([[0]], cuda), ints([n], cuda), 1.0)
    k = decode(rows, d)
    p = torch.softmax(q.double().cpu().view(1, d) @ k.t(), -1)
    assert rel(out.view(1, d), p @ k) <= bar(torch.float16)


# --- Capped and biased scores over the other caches --------------------------------------------------


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("types", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")],
                         ids="-".join)
@pytest.mark.parametrize("cap", [0.3, 6.0, 50.0])
@pytest.mark.parametrize("wide", [False, True], ids=["narrow", "wide"])
def test_scores_over_plain_caches(cuda, types, d, cap, wide):
    """Caps that all, some and no scores come near, with and without slopes; a sequence's last page cut."""
    from test_paged_gpu import Cache

    dt, ct = (TYPES[t] for t in types)
    lengths = [1, 16, 33, 0, 129, 511] + ([2500] if wide else [])
    c = Cache(cuda, ct, 2, 32, d, lengths, seed=10)
    q = q_of(cuda, dt, len(lengths), 4, d, spread=4.0)
    for slopes in (None, torch.tensor([0.5, 0.0, -0.002, 3.0], device=cuda)):
        out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5, cap=cap, slopes=slopes)
        ref, top = attended(q, c, lengths, d ** -0.5, cap, slopes)
        assert rel(out, ref) <= bar(dt, max(top, 10.0)), slopes


def test_scores_infinite_keys(cuda):
    """Infinite scores stay within the cap: their keys weigh what the cap gives them."""
    from test_paged_gpu import Cache

    c = Cache(cuda, torch.float32, 1, 16, 32, [20], seed=11)
    c.k[int(c.table[0, 0]), 0, 3, 0] = float("inf")
    q = q_of(cuda, torch.float32, 1, 2, 32)
    q[0, 0, 0, 0], q[0, 1, 0, 0] = 1.0, -1.0
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.2, cap=3.0)
    ref, top = attended(q, c, [20], 0.2, 3.0)
    assert bool(ref.isfinite().all()) and rel(out, ref) <= bar(torch.float32, top)


# --- Readings ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "fp4"])
@pytest.mark.parametrize("to", [None, "f32", "f16", "bf16"])
def test_read(cuda, cache, to, d):
    """Ragged windows, before the first and behind the last token, pages that are missing."""
    from test_paged_gpu import Cache

    lengths, starts, s = [70, 0, 33, 100, 5], [60, 0, -4, 0, 7], 50
    c = Four(cuda, 3, 16, d, lengths, seed=12) if cache == "fp4" else Cache(cuda, TYPES[cache], 3, 16, d, lengths, seed=12)
    table = c.table.clone()
    table[3, 2], table[2, 1] = 10 ** 6, -1
    native = torch.bfloat16 if cache == "fp4" else TYPES[cache]
    dt = TYPES[to] if to else native
    k, v = cfa.paged_read(c.k, c.v, table, c.lengths, s, starts=ints(starts, cuda), dtype=TYPES[to] if to else None)
    for got, which in ((k, 0), (v, 1)):
        want = torch.zeros(5, 3, s, d, dtype=torch.float64)
        for i, (n, first) in enumerate(zip(lengths, starts)):
            dense = c.dense(i, n)[which] if n else None
            for j in range(s):
                t = first + j
                if 0 <= t < n:
                    gone = (i == 3 and t // 16 == 2) or (i == 2 and t // 16 == 1)
                    want[i, :, j] = float("nan") if gone else dense[:, t]
        assert got.dtype == dt and got.is_contiguous() and got.shape == want.shape
        assert torch.equal(got.cpu().nan_to_num(9.0), want.to(dt).nan_to_num(9.0))
        assert torch.equal(got.cpu().isnan(), want.isnan())
    k0, _ = cfa.paged_read(c.k, c.v, c.table, c.lengths, 3)
    assert torch.equal(k0[0, 1].double().cpu(), c.dense(0, 3)[0][1])
    assert cfa.paged_read(c.k, c.v, c.table, c.lengths, 0)[0].shape == (5, 3, 0, d)


def test_read_past_the_table(cuda):
    """A length that the table has no room for: NaN from its end on."""
    c = Four(cuda, 1, 16, 32, [32], seed=13)
    k, v = cfa.paged_read(c.k, c.v, c.table, ints([40], cuda), 50)
    assert not bool(k[:, :, :32].isnan().any()) and bool(k[:, :, 32:40].isnan().all() and v[:, :, 32:40].isnan().all())
    assert float(k[:, :, 40:].abs().max()) == 0.0


def test_far_pages(cuda):
    """A pool of more than 2^32 bytes, its last pages in use: as a small pool, bit for bit."""
    far = torch.empty(2, 130000, 8, 64, 36, dtype=torch.uint8, device=cuda)
    near = torch.zeros(2, 3, 8, 64, 36, dtype=torch.uint8, device=cuda)
    far[:, -3:] = 0
    gen = torch.Generator().manual_seed(14)
    k, v = (torch.randn(1, 8, 130, 64, generator=gen).bfloat16().to(cuda) for _ in range(2))
    q = q_of(cuda, torch.bfloat16, 1, 16, 64, seed=19)
    out = []
    for pool, first in ((far, 129997), (near, 0)):
        table = ints([[first + 2, first, first + 1]], cuda)
        cfa.paged_append(k, v, pool[0], pool[1], table, ints([0], cuda))
        out.append((cfa.paged_attention(q, pool[0], pool[1], table, ints([130], cuda), 0.125),
                    *cfa.paged_read(pool[0], pool[1], table, ints([130], cuda), 130)))
    assert torch.equal(far[:, -3:], near) and all(torch.equal(x, y) for x, y in zip(*out))
    assert float(out[0][0].abs().max()) > 0


# --- Together ---------------------------------------------------------------------------------------


def test_decoding_step_captured(cuda):
    """A decoding step over 4 bits in a graph, replayed with other tokens, lengths and tables in the same
    buffers, eager work between: each replay equals the eager calls bit for bit."""
    b, h, hk, d = 3, 4, 2, 64
    c = Four(cuda, hk, 16, d, [900, 40, 0], room=32, seed=15)
    f = cfa.rotary_frequencies(d, device=cuda)
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4], device=cuda)
    q, k, v = (torch.randn(b, n, 1, d, device=cuda).bfloat16() for n in (h, hk, hk))
    lengths = c.lengths.clone()

    def step(kp, vp, lengths):
        qt = cfa.paged_append(k, v, kp, vp, c.table, lengths, q=q, frequencies=f)
        before = lengths.clone()
        lengths.add_(1)
        out = cfa.paged_attention(qt, kp, vp, c.table, lengths, 0.125, cap=5.0, slopes=slopes)
        return [out, *cfa.paged_read(kp, vp, c.table, lengths, 1, starts=before)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kp, vp = c.k.clone(), c.v.clone()
    with torch.cuda.stream(side):
        step(kp.clone(), vp.clone(), lengths.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(kp, vp, lengths)
    ek, ev, el = c.k.clone(), c.v.clone(), c.lengths.clone()
    kp.copy_(c.k), vp.copy_(c.v), lengths.copy_(c.lengths)
    for i in range(4):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        graph.replay()
        out = [x.clone() for x in got]
        want = step(ek, ev, el)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i
    assert torch.equal(kp, ek) and torch.equal(vp, ev) and torch.equal(lengths, el)


def test_two_calls_in_flight(cuda):
    """Two batches on two streams, each call with a workspace of its own, an append before each on its stream."""
    caches = [Four(cuda, 2, 16, 64, [3000, 40, 1700], room=8, seed=30 + i) for i in range(2)]
    q = [q_of(cuda, torch.bfloat16, 3, 8, 64, seed=40 + i) for i in range(2)]
    k = [torch.randn(3, 2, 8, 64, generator=torch.Generator().manual_seed(50 + i)).bfloat16().to(cuda) for i in range(2)]
    start = [(c.k.clone(), c.v.clone()) for c in caches]

    def step(i, kp, vp):
        c = caches[i]
        cfa.paged_append(k[i], k[i], kp, vp, c.table, c.lengths)
        return [cfa.paged_attention(q[i], kp, vp, c.table, c.lengths + 8, 0.125, cap=20.0),
                *cfa.paged_read(kp, vp, c.table, c.lengths + 8, 64, starts=c.lengths - 30)]

    want = [step(i, caches[i].k, caches[i].v) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i, *start[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for i in range(2) for out in got[i] for x, y in zip(out, want[i]))


def test_saved_pages_refuse_their_backward(cuda):
    """An append of codes counts as a write of the pages, as the others do."""
    c = Four(cuda, 1, 16, 32, [3], room=2, seed=16)
    before = (c.k._version, c.v._version)
    k = torch.randn(1, 1, 2, 32, device=cuda)
    cfa.paged_append(k, k, c.k, c.v, c.table, c.lengths)
    assert c.k._version > before[0] and c.v._version > before[1]


def test_refusals_on_the_device(cuda):
    c = Four(cuda, 2, 16, 64, [3], seed=17)
    q = q_of(cuda, torch.float32, 1, 2, 64)
    x = torch.zeros(1, 2, 1, 64, device=cuda)
    slopes = torch.zeros(2, device=cuda)
    for call, text in [
        (lambda: cfa.paged_append(x, x, c.k, c.k, c.table, c.lengths), "same memory"),
        (lambda: cfa.paged_append(x, x, c.k[..., :32], c.v[..., :32], c.table, c.lengths), "36"),
        (lambda: cfa.paged_append(x, x, c.k, c.v.float(), c.table, c.lengths), "must be uint8"),
        (lambda: cfa.paged_attention(x[..., :32].contiguous(), c.k, c.v, c.table, c.lengths, 1.0), "20"),
        (lambda: cfa.paged_attention(q, c.k[..., 1:33], c.v[..., 1:33], c.table, c.lengths, 1.0), "36"),
        (lambda: cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 1.0, cap=1e31), "cap"),
        (lambda: cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 1.0, slopes=slopes[:1]), "slopes"),
        (lambda: cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 1.0, slopes=slopes.double()), "float32"),
        (lambda: cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 1.0, slopes=slopes.cpu()), "HIP device"),
        (lambda: cfa.paged_read(c.k, c.v, c.table, c.lengths, -1), "number of tokens"),
        (lambda: cfa.paged_read(c.k, c.v, c.table, c.lengths, 1, starts=c.lengths.long()), "int32"),
        (lambda: cfa.paged_read(c.k[..., :33], c.v[..., :33], c.table, c.lengths, 1), "expected"),
    ]:
        with pytest.raises(cfa.FusedAttentionError, match=text):
            call()
    buf = torch.zeros(c.k.numel() + 2, dtype=torch.uint8, device=cuda)
    off = buf[2:].view(c.k.shape)
    with pytest.raises(cfa.FusedAttentionError, match="4-byte aligned"):
        cfa.paged_attention(q, off, c.v, c.table, c.lengths, 1.0)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,dim", [(64, 8), (64, 16), (64, 40), (64, 48), (64, 56), (128, 8), (128, 16), (128, 72),
                                   (128, 80), (128, 96), (128, 120)])
def test_append_partly_turned_groups(cuda, d, dim, dtype, interleaved):
    """Turned and other values under one scale: alike, one part 50 times the other, one of zeros, a NaN or an
    infinity in one part; the same bytes for a token alone, whose neighbours leave nothing in doubt."""
    dt, n = TYPES[dtype], 24
    gen = torch.Generator().manual_seed(d + dim)
    k = torch.randn(7, 2, n, d, generator=gen)
    k[1, ..., :dim] *= 50.0
    k[2, ..., dim:] *= 50.0
    k[3, ..., :dim] = 0.0
    k[4, ..., dim:] = 0.0
    k[5, :, ::2, dim], k[5, :, 1::2, dim - 1] = float("nan"), float("nan")
    k[6, :, ::2, dim], k[6, :, 1::2, dim - 1] = float("inf"), -float("inf")
    k = k.to(dt)
    v = torch.randn(7, 2, n, d, generator=gen).to(dt)
    f = cfa.rotary_frequencies(dim, device=cuda)
    table = torch.arange(14, dtype=torch.int32, device=cuda).view(7, 2)
    held = ints([0, 1, 2, 3, 4, 5, 6], cuda)
    kp, vp, k1, v1 = (torch.zeros(14, 2, 16, cfa.fp4_row_bytes(d), dtype=torch.uint8, device=cuda) for _ in range(4))
    cfa.paged_append(k.to(cuda), v.to(cuda), kp, vp, table, held, frequencies=f, interleaved=interleaved)
    got_k, got_v = (x.view(7, 2, 2, 16, -1).transpose(1, 2).flatten(2, 3).cpu() for x in (kp, vp))
    for i in range(7):
        want = encode(turned(k[i], torch.arange(i, i + n), f, interleaved))
        assert torch.equal(got_k[i, :, i:i + n], want), i
        assert torch.equal(got_v[i, :, i:i + n], encode(v[i])), i
    for t in range(n):
        cfa.paged_append(k[:, :, t:t + 1].to(cuda), v[:, :, t:t + 1].to(cuda), k1, v1, table, held + t, frequencies=f,
                         interleaved=interleaved)
    assert torch.equal(kp, k1) and torch.equal(vp, v1)


def codes_under(byte):
    """A row of 32: every code twice, in order and back, under one scale byte."""
    row = torch.zeros(20, dtype=torch.uint8)
    codes = list(range(16)) + list(range(15, -1, -1))
    row[:16] = torch.tensor([x | y << 4 for x, y in zip(codes[0::2], codes[1::2])], dtype=torch.uint8)
    row[16] = byte
    return row


BYTES = [0, 1, 2, 64, 126, 127, 128, 252, 253, 254, 255]


def same(x, y):
    """Equal, infinities by their sign, NaN where the other is."""
    x, y = x.cpu(), y.cpu()
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x[~x.isnan()], y[~y.isnan()])


@pytest.mark.parametrize("to", TYPES)
def test_read_every_code_at_the_ends(cuda, to):
    """Scales from 2^-127 on (subnormal values) to 2^127, past which codes are infinities, and NaN."""
    kp = torch.zeros(1, 1, 16, 20, dtype=torch.uint8)
    kp[0, 0, :len(BYTES)] = torch.stack([codes_under(x) for x in BYTES])
    vp = kp.flip(2)
    n = len(BYTES)
    k, v = cfa.paged_read(kp.to(cuda), vp.to(cuda), ints([[0]], cuda), ints([16], cuda), 16, dtype=TYPES[to])
    ref = decode(kp[0, 0], 32).float().to(TYPES[to])
    assert bool(ref[BYTES.index(253)].isinf().any()) and bool(ref[n - 1].isnan().all())
    assert same(k[0, 0], ref) and same(v[0, 0], ref.flip(0))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_values_at_the_ends(cuda, dtype, d):
    """One token's weight is 1, whose lower terms are 0: its values come back, infinities among them. (Of type f16
    or bf16 rounded once.) In a longer sequence they leave the other 32 head_dims as they are."""
    n = len(BYTES)
    rows = torch.zeros(n, 1, 16, cfa.fp4_row_bytes(d), dtype=torch.uint8)
    for i, byte in enumerate(BYTES):
        row = codes_under(byte)
        for g in range(d // 32):
            rows[i, 0, 0, 16 * g:16 * (g + 1)] = row[:16]
            rows[i, 0, 0, d // 2 + g] = byte if g == 0 else 127
    kp = torch.zeros_like(rows)
    kp[..., d // 2:d // 2 + d // 32] = 127
    table = torch.arange(n, dtype=torch.int32, device=cuda)[:, None]
    q = q_of(cuda, TYPES[dtype], n, 1, d)
    out = cfa.paged_attention(q, kp.to(cuda), rows.to(cuda), table, ints([1] * n, cuda), 1.0)
    ref = decode(rows[:, 0, 0], d).float().to(TYPES[dtype])
    for i, byte in enumerate(BYTES):
        if byte > 2:
            assert same(out[i, 0, 0], ref[i]), (byte, out[i, 0, 0], ref[i])
        else:  # (values below the least normal float: products may flush them)
            assert float((out[i, 0, 0].double().cpu() - ref[i].double()).abs().max()) <= 2.0 ** -126
    c = Four(cuda, 2, 16, d, [300, 700], seed=18)
    q = q_of(cuda, TYPES[dtype], 2, 4, d)
    clean = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, d ** -0.5)
    for byte, code in ((253, 6), (253, 15), (254, 4), (254, 13)):
        v = c.v.clone()
        row = v[int(c.table[1, 20]), 1, 3]
        row[:16], row[d // 2] = code | code << 4, byte
        out = cfa.paged_attention(q, c.k, v, c.table, c.lengths, d ** -0.5)
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :2], clean[1, :2])
        assert torch.equal(out[1, 2:, :, 32:], clean[1, 2:, :, 32:])
        want = -float("inf") if code & 8 else float("inf")
        assert bool((out[1, 2:, :, :32] == want).all())


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_append_keys_past_the_largest_float(cuda, interleaved):
    """Turned past the largest float, a key counts as it; a value from 3.5 x 2^126 on is stored as 4 x 2^126."""
    big = torch.finfo(torch.float32).max
    k = torch.full((1, 1, 3, 64), 3e38)
    k[..., 1::2] = -2.9e38
    k[0, 0, 2] = torch.linspace(-1.0, 1.0, 64) * big
    f = torch.full((32,), 0.7, dtype=torch.float64, device=cuda)
    kp, vp = (torch.zeros(1, 1, 16, 36, dtype=torch.uint8, device=cuda) for _ in range(2))
    cfa.paged_append(k.to(cuda), k.to(cuda), kp, vp, ints([[0]], cuda), ints([1], cuda), frequencies=f,
                     interleaved=interleaved)
    y = turned(k[0], torch.arange(1, 4), f, interleaved)
    assert float(y.abs().max()) > big
    assert torch.equal(kp[0, :, 1:4].cpu(), encode(y.clamp(-big, big)))
    assert torch.equal(vp[0, :, 1:4].cpu(), encode(k[0]))


@pytest.mark.parametrize("cap", [None, 3.0], ids=["plain", "capped"])
def test_attention_slopes_to_the_largest_float(cuda, cap):
    """Slopes that are floats but not in units of log2 e, or not times a distance: the last token alone."""
    lengths = [1, 2, 33, 700, 3000]
    c = Four(cuda, 2, 16, 64, lengths, seed=19)
    q = q_of(cuda, torch.float32, len(lengths), 4, 64)
    slopes = torch.tensor([torch.finfo(torch.float32).max, 2.4e38, 1e38, 1e37], device=cuda)
    out = cfa.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, cap=cap, slopes=slopes)
    ref, _ = attended(q, c, lengths, 0.125, cap, slopes)
    assert rel(out, ref) <= bar(torch.float32)


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("d,dim", [(32, 32), (64, 64), (64, 40), (128, 128)])
@pytest.mark.parametrize("magnitude,spread", [(1e-42, 1e30), (1e-45, 1e37), (1e-38, 1e30), (1e-31, 1e30), (0.0, 1.0),
                                              (-1.0, 1.0), (1e30, 1e-30)])
def test_append_magnitudes(cuda, d, dim, magnitude, spread, interleaved):
    """Magnitudes that 32 bits hold with few bits or as 0, of keys that make up for them; 0, and a negative one."""
    k = torch.randn(1, 2, 60, d, generator=torch.Generator().manual_seed(d)) * spread
    k[..., dim:] /= spread
    f = cfa.rotary_frequencies(dim, device=cuda)
    kp, vp = (torch.zeros(4, 2, 16, cfa.fp4_row_bytes(d), dtype=torch.uint8, device=cuda) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=cuda)[None]
    cfa.paged_append(k.to(cuda), k.to(cuda), kp, vp, table, ints([1], cuda), frequencies=f, interleaved=interleaved,
                     magnitude=magnitude)
    got_k, got_v = (x.transpose(0, 1).flatten(1, 2)[:, 1:61].cpu() for x in (kp, vp))
    assert torch.equal(got_k, encode(turned(k[0], torch.arange(1, 61), f, interleaved, magnitude)))
    assert torch.equal(got_v, encode(k[0]))
