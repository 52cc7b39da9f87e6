"""Timed workloads of attention with scores of other forms, and of the paged cache in 4 bits, called as a
user's program calls them.

A case is one call pattern. `op` names the operator:
  scored      fused_scored_attention of the last sq of sk positions: scores capped ("cap", 0: not),
              lowered by a slope times the distance ("slopes"), masked causally, by documents ("docs":
              their mean length, 0: one) with padding behind them ("pad"), and with a prefix that every
              query sees ("prefix", the longest of the batch); with "train" the backward too;
  paged       paged_attention of one token per sequence over lo .. hi cached tokens, with the same cap
              and slopes;
  append      paged_append of `s` new tokens (ragged with "ragged") to 4-bit caches that hold lo .. hi
              tokens, keys and queries rotated on the way, and paged_read of what the cache then has of
              them;
  read        paged_read of `s` tokens per sequence of lo .. hi.
Inputs are N(0, 1), the queries of capped scores N(0, 9) (trained models' scores come near their cap),
scale 1 / sqrt(d). Types: `dtype` is the activations', `cache` the cache's ("fp4": 4 bits).

With `own` false the same results come from elementary torch operations in 32 bits (what is next to a
border, and angles, in 64).
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
_PKG = str(Path(__file__).resolve().parent.parent / "candle-fused-attn_amd")
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp4": torch.uint8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import candle_fused_attn
    return candle_fused_attn


def listed():
    return [
        # One short sequence's training step, one layer: latency.
        {"name": "scored_short_train", "op": "scored", "b": 1, "h": 6, "hk": 6, "sq": 240, "sk": 240,
         "d": 64, "causal": True, "cap": 30.0, "slopes": False, "docs": 0, "pad": 0, "prefix": 0,
         "train": True},
        # A training step on packed documents, some samples padded.
        {"name": "scored_packed_train", "op": "scored", "b": 8, "h": 12, "hk": 12, "sq": 2048,
         "sk": 2048, "d": 64, "causal": True, "cap": 50.0, "slopes": False, "docs": 600, "pad": 200,
         "prefix": 0, "train": True},
        # Wide heads in groups, a bias by distance, prompts that see themselves whole, an odd length.
        {"name": "scored_prefix_train", "op": "scored", "b": 4, "h": 16, "hk": 4, "sq": 777, "sk": 777,
         "d": 128, "causal": True, "cap": 0.0, "slopes": True, "docs": 0, "pad": 0, "prefix": 200,
         "train": True},
        # The next chunk of two long prompts, over all that came before it.
        {"name": "scored_chunk", "op": "scored", "b": 2, "h": 32, "hk": 8, "sq": 512, "sk": 4097,
         "d": 128, "causal": True, "cap": 0.0, "slopes": True, "docs": 0, "pad": 0, "prefix": 0,
         "train": False},
        # One new token of one short sequence, fp32 throughout: latency.
        {"name": "capped_one", "op": "paged", "b": 1, "h": 6, "hk": 6, "d": 64, "dtype": "f32",
         "cache": "f32", "page": 16, "lo": 240, "hi": 240, "cap": 30.0, "slopes": False},
        # A serving batch of unequal sequences.
        {"name": "capped_batch", "op": "paged", "b": 64, "h": 6, "hk": 6, "d": 64, "dtype": "bf16",
         "cache": "bf16", "page": 16, "lo": 1, "hi": 2048, "cap": 50.0, "slopes": True},
        # One decoding step of a batch: one token each into 4-bit caches of any fill.
        {"name": "four_append_token", "op": "append", "b": 64, "h": 6, "hk": 6, "s": 1, "d": 64,
         "dim": 64, "dtype": "f32", "page": 16, "lo": 1, "hi": 1000, "interleaved": False,
         "ragged": False},
        # The prompts of a batch, padded to the longest, into empty 4-bit caches.
        {"name": "four_append_prompts", "op": "append", "b": 16, "h": 32, "hk": 8, "s": 2048, "d": 128,
         "dim": 128, "dtype": "bf16", "page": 64, "lo": 0, "hi": 0, "interleaved": False,
         "ragged": True},
        # The batch of unequal sequences over 4-bit caches, fp32 activations.
        {"name": "four_batch", "op": "paged", "b": 64, "h": 6, "hk": 6, "d": 64, "dtype": "f32",
         "cache": "fp4", "page": 16, "lo": 1, "hi": 2048, "cap": 0.0, "slopes": False},
        # Few very long contexts in 4 bits, grouped wide heads.
        {"name": "four_long", "op": "paged", "b": 4, "h": 32, "hk": 8, "d": 128, "dtype": "bf16",
         "cache": "fp4", "page": 64, "lo": 60000, "hi": 131071, "cap": 0.0, "slopes": True},
        # The last chunk of a few sequences back out of the cache, narrow heads.
        {"name": "read_chunk", "op": "read", "b": 5, "hk": 12, "s": 333, "d": 32, "dtype": "f16",
         "cache": "f16", "page": 32, "lo": 100, "hi": 1000},
        # Long contexts out of a 4-bit cache, for a chunk's attention over them.
        {"name": "read_context", "op": "read", "b": 4, "hk": 8, "s": 32767, "d": 128, "dtype": "bf16",
         "cache": "fp4", "page": 64, "lo": 20000, "hi": 40000},
    ]


def _cost(case):
    """What bounds a pass of either form: bytes, operations, and the scores that a dense form holds."""
    w = work(case)
    dense = case["b"] * case["h"] * case["sq"] * case["sk"] if case["op"] == "scored" else 0
    return w["bytes"], w["flops"], dense


_MOST = None


def _most():
    """The most a drawn case may cost, by operator: the largest listed one's."""
    global _MOST
    if _MOST is None:
        _MOST = {}
        for case in listed():
            at = _MOST.get(case["op"], (0, 0, 0))
            _MOST[case["op"]] = tuple(max(x, y) for x, y in zip(at, _cost(case)))
    return _MOST


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hk = rng.choice((1, 2, 3, 4, 6, 8))
    return hk * rng.choice((1, 1, 2, 3, 4, 8)), hk


def _draw(rng):
    op = rng.choice(("scored", "scored", "paged", "paged", "append", "read"))
    h, hk = _heads(rng)
    d = rng.choice((32, 64, 64, 128))
    page = rng.choice((16, 32, 48, 64, 128))
    cap = rng.choice((0.0, 0.0, 5.0, 20.0, 50.0))
    dtype, cache = rng.choice((("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                               ("bf16", "bf16"), ("f32", "fp4"), ("f16", "fp4"), ("bf16", "fp4")))
    if op == "scored":
        sk = _log(rng, 1, 4097)
        causal = rng.random() < 0.7
        return {"op": op, "b": _log(rng, 1, 64), "h": h, "hk": hk,
                "sq": rng.choice((sk, sk, _log(rng, 1, sk))), "sk": sk, "d": d, "causal": causal,
                "cap": cap, "slopes": rng.random() < 0.5,
                "docs": rng.choice((0, _log(rng, 1, sk))), "pad": rng.choice((0, 0, sk // 3)),
                "prefix": rng.choice((0, sk // 4)) if causal else 0, "train": rng.random() < 0.6}
    if op == "paged":
        hi = _log(rng, 1, 131071)
        return {"op": op, "b": _log(rng, 1, 128), "h": h, "hk": hk, "d": d, "dtype": dtype,
                "cache": cache, "page": page, "lo": rng.choice((0, 1, hi // 2, hi)), "hi": hi,
                "cap": cap, "slopes": rng.random() < 0.5 or (cap == 0.0 and cache != "fp4")}
    if op == "append":
        s = rng.choice((1, _log(rng, 2, 2048)))
        return {"op": op, "b": _log(rng, 1, 64), "h": h, "hk": hk, "s": s, "d": d,
                "dim": rng.choice((d, d, d // 2)), "dtype": dtype, "page": page, "lo": 0,
                "hi": rng.choice((0, _log(rng, 1, 4096))), "interleaved": rng.random() < 0.5,
                "ragged": s > 1 and rng.random() < 0.7}
    hi = _log(rng, 1, 40000)
    return {"op": op, "b": _log(rng, 1, 64), "hk": hk, "s": _log(rng, 1, hi), "d": d,
            "dtype": rng.choice(("f32", "bf16", "f16")) if cache == "fp4" else cache, "cache": cache,
            "page": page, "lo": rng.choice((0, hi // 2, hi)), "hi": hi}


def _telling(case):
    """Whether a gradient is more than the rounding of a zero (a query that sees one key has none)."""
    return not case.get("train") or _pairs(case) >= 1.5 * case["b"] * case["sq"]


def draw(rng):
    while True:
        case = _draw(rng)
        if _telling(case) and all(x <= y for x, y in zip(_cost(case), _most()[case["op"]])):
            return case


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def _lengths(b, lo, hi):
    """b lengths spread evenly from hi down to lo (the first is hi): the same for every seed."""
    return [hi - (hi - lo) * i // max(b - 1, 1) for i in range(b)]


def _counts(case):
    """New tokens of each sequence of an append."""
    return _lengths(case["b"], max(1, case["s"] // 3), case["s"]) if case["ragged"] else (
        [case["s"]] * case["b"])


def _held(case):
    """Tokens each sequence's cache holds before an append, or has for an attention or a reading."""
    return _lengths(case["b"], case["lo"], case["hi"])


def _spans(case):
    """Each sample's documents, (first, behind the last) one after the other from 0 on; what they leave
    of sk is padding. Their lengths are 0.4 to 1.6 of the mean, the same for every seed."""
    out = []
    for i, pad in enumerate(_lengths(case["b"], 0, case["pad"])):
        end, at, spans, x = case["sk"] - pad, 0, [], 7919 * (i + 1)
        while at < end:
            x = (1103515245 * x + 12345) % (1 << 31)
            n = end if case["docs"] == 0 else max(1, case["docs"] * (400 + (x >> 8) % 1201) // 1000)
            spans.append((at, min(at + n, end)))
            at += n
        out.append(spans)
    return out


def _prefixes(case):
    return _lengths(case["b"], 0, case["prefix"])


def _masked(case):
    return case["docs"] > 0 or case["pad"] > 0


def _pairs(case):
    """The (query, key) pairs that the masks let through, of one head over the whole batch."""
    total = 0
    for spans, prefix in zip(_spans(case), _prefixes(case)):
        for first, end in spans:
            i = np.arange(max(first, case["sk"] - case["sq"]), end)
            if case["causal"]:
                total += int((np.maximum(i + 1, min(prefix, end)) - first).sum())
            else:
                total += len(i) * (end - first)
    return total


def _frequencies(dim):
    """Radians per position of each of a head's dim / 2 pairs, 10000^(-2 i / dim)."""
    return (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).to(DEVICE)


def _slopes(case):
    """2^(-8 (i + 1) / h) of head i."""
    i = torch.arange(1, case["h"] + 1, dtype=torch.float32)
    return torch.exp2(-8.0 * i / case["h"]).to(DEVICE) if case["slopes"] else None


def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(_TYPES[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def _row(d):
    """Bytes of d values in 4 bits: two to a byte, a scale byte per 32, up to a multiple of 4."""
    return d // 2 + 4 * max(1, d // 128)


def _pages(gen, case, lengths, most):
    """A page pool with `most` tokens' room for the longest sequence, and a table that deals its pages
    out in random order."""
    per = [-(-n // case["page"]) for n in lengths]
    wide = max(1, -(-most // case["page"]))
    order = torch.randperm(max(1, sum(per)), generator=gen, device=DEVICE).to(torch.int32)
    rows = torch.zeros(case["b"], wide, dtype=torch.int32, device=DEVICE)
    at = torch.arange(wide, device=DEVICE)[None, :] < _ints(per)[:, None]
    rows[at] = order[:sum(per)]
    shape = (max(1, sum(per)), case["hk"], case["page"], case["d"])
    pools = []
    for _ in range(2):
        if case["cache"] == "fp4":
            pools.append(torch.cat([_encode(_normal(gen, "f32", len(x), *shape[1:]))
                                    for x in torch.arange(shape[0]).split(4096)]))
        else:
            pools.append(_normal(gen, case["cache"], *shape))
    return *pools, rows


def _scored_inputs(case, seed):
    gen, b, d, sq, sk = _generator(seed), case["b"], case["d"], case["sq"], case["sk"]
    q, g = (_normal(gen, "f32", b, sq, case["h"], d).transpose(1, 2) for _ in range(2))
    k, v = (_normal(gen, "f32", b, sk, case["hk"], d).transpose(1, 2) for _ in range(2))
    st = {"q": q * 3.0 if case["cap"] else q, "k": k, "v": v, "g": g if case["train"] else None,
          "cap": case["cap"] or None, "slopes": _slopes(case), "documents": None, "prefix": None}
    if _masked(case):
        ids = np.full((b, sk), -1, dtype=np.int32)
        for row, spans in zip(ids, _spans(case)):
            for n, (first, end) in enumerate(spans):
                row[first:end] = n
        st["documents"] = torch.from_numpy(ids).to(DEVICE)
    if case["prefix"]:
        st["prefix"] = _ints(_prefixes(case))
    return st


def _paged_inputs(case, seed):
    gen, lengths = _generator(seed), _held(case)
    kp, vp, table = _pages(gen, case, lengths, max(lengths))
    q = _normal(gen, "f32", case["b"], case["h"], 1, case["d"]) * (3.0 if case["cap"] else 1.0)
    return {"q": q.to(_TYPES[case["dtype"]]), "k_pages": kp, "v_pages": vp, "table": table,
            "lengths": _ints(lengths), "cap": case["cap"] or None, "slopes": _slopes(case)}


def _append_inputs(case, seed):
    gen, b, s, d = _generator(seed), case["b"], case["s"], case["d"]
    held, counts = _held(case), _counts(case)
    total = [x + y for x, y in zip(held, counts)]
    kp, vp, table = _pages(gen, {**case, "cache": "fp4"}, total, max(total))
    q, k, v = (_normal(gen, case["dtype"], b, s, n, d).transpose(1, 2)
               for n in (case["h"], case["hk"], case["hk"]))
    return {"q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, "table": table,
            "lengths": _ints(held), "after": _ints(total),
            "counts": _ints(counts) if case["ragged"] else None, "frequencies": _frequencies(case["dim"])}


def _read_inputs(case, seed):
    """The last `s` tokens of each sequence; a shorter one is read from its beginning."""
    gen, lengths = _generator(seed), _held(case)
    kp, vp, table = _pages(gen, case, lengths, max(lengths))
    return {"k_pages": kp, "v_pages": vp, "table": table, "lengths": _ints(lengths),
            "starts": _ints([max(0, n - case["s"]) for n in lengths])}


_INPUTS = {"scored": _scored_inputs, "paged": _paged_inputs, "append": _append_inputs,
           "read": _read_inputs}


def prepare(case, seed):
    state = _INPUTS[case["op"]](case, seed)
    if case.get("train"):
        for t in ("q", "k", "v"):
            state[t].requires_grad_(True)
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------
# Values in 4 bits: a sign and a magnitude of 0, .5, 1, 1.5, 2, 3, 4 or 6, times a power of two that 32
# values share, the least one under which none of them passes 7
# ------------------------------------------------------------------------------------------------


def _encode(x):
    """x [..., d] as bytes [..., _row(d)]: codes, the first of two in the low bits (the nearest
    magnitude, the even code between two; no negative zero), then the scales' exponents + 127, 255 for
    values of which one is not finite. Exact in x's own type."""
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    m, e = torch.frexp(top)
    e = (e - 3 + (m > 0.875)).clamp_min(-127).masked_fill(top == 0, -127)
    fine = top.isfinite()
    e = e.masked_fill(~fine, 0)
    u = torch.ldexp(g.abs(), -e[..., None])
    code = ((u > 0.25).byte() + (u >= 0.75).byte() + (u > 1.25).byte() + (u >= 1.75).byte()
            + (u > 2.5).byte() + (u >= 3.5).byte() + (u > 5.0).byte())
    code = torch.where((g < 0) & (code > 0), code + 8, code) * fine[..., None]
    code = code.flatten(-2)
    scale = torch.where(fine, e + 127, 255).byte()
    pad = torch.zeros(*x.shape[:-1], -scale.shape[-1] % 4, dtype=torch.uint8, device=x.device)
    return torch.cat((code[..., 0::2] | (code[..., 1::2] << 4), scale, pad), dim=-1)


def _decode(rows, d):
    """The values of bytes [..., _row(d)], in 32 bits."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=rows.device)
    levels = torch.cat((levels, -levels))
    powers = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], device=rows.device)
    pairs = rows[..., :d // 2]
    codes = torch.stack((pairs & 15, pairs >> 4), dim=-1).flatten(-2)
    scales = powers[rows[..., d // 2:d // 2 + d // 32].int()]
    return (levels[codes.int()].unflatten(-1, (-1, 32)) * scales[..., None]).flatten(-2)


def _cached(rows, d):
    """What a cache's rows hold, in 32 bits."""
    return _decode(rows, d) if rows.dtype == torch.uint8 else rows.float()


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """x [b, h, s, d] rotated by angles [b, 1, s, dim / 2], in the angles' type."""
    x, n = x.to(cos.dtype), cos.shape[-1]
    if interleaved:
        a, c = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * cos - c * sin, c * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, c = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * cos - c * sin, c * cos + a * sin), dim=-1)
    return torch.cat((y, x[..., 2 * n:]), dim=-1)


def _softmax(scores, mask):
    """Softmax over the last dimension where `mask` holds; rows that it leaves empty are 0."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _visible(state):
    """[b, 1, sq, sk] (or 1 in b's place): who sees whom."""
    case = state["case"]
    j = torch.arange(case["sk"], device=DEVICE)
    i = j[case["sk"] - case["sq"]:, None]
    seen = torch.ones(1, 1, case["sq"], case["sk"], dtype=torch.bool, device=DEVICE)
    if case["causal"]:
        seen = (j <= i)[None, None]
        if state["prefix"] is not None:
            seen = seen | (j < state["prefix"][:, None, None, None])
    if state["documents"] is not None:
        ids = state["documents"][:, None, None, :]
        mine = ids[..., case["sk"] - case["sq"]:].transpose(2, 3)
        seen = seen & (ids == mine) & (mine >= 0)
    return seen


def _run_scored(state):
    case = state["case"]
    scale = 1.0 / math.sqrt(case["d"])
    leaves = [state["q"], state["k"], state["v"]]
    if own:
        cfa = _framework()

        def forward():
            return cfa.fused_scored_attention(*leaves, scale, case["causal"], cap=state["cap"],
                                              slopes=state["slopes"], documents=state["documents"],
                                              prefix=state["prefix"])

        if not case["train"]:
            with torch.no_grad():
                return [forward()]
        out = forward()
        return [out.detach(), *torch.autograd.grad(out, leaves, state["g"])]
    with torch.no_grad():
        b, h, hk, sq, sk, d = (case[n] for n in ("b", "h", "hk", "sq", "sk", "d"))
        q = leaves[0].reshape(b, hk, h // hk * sq, d)
        k, v = (t.contiguous() for t in leaves[1:])
        x = torch.matmul(q, k.transpose(2, 3)) * scale
        if case["cap"]:
            t = torch.tanh(x / case["cap"])
            x = case["cap"] * t
        x = x.view(b, h, sq, sk)
        if state["slopes"] is not None:
            j = torch.arange(sk, device=DEVICE, dtype=torch.float32)
            x = x - state["slopes"][:, None, None] * (j[sk - sq:, None] - j).abs()
        p = _softmax(x, _visible(state)).view(b, hk, h // hk * sq, sk)
        o = torch.matmul(p, v)
        out = [o.view(b, h, sq, d)]
        if case["train"]:
            g = state["g"].reshape(b, hk, h // hk * sq, d)
            ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * o).sum(-1, keepdim=True)) * scale
            if case["cap"]:
                ds = ds * (1.0 - t * t)
            out += [torch.matmul(ds, k).view(b, h, sq, d), torch.matmul(ds.transpose(2, 3), q),
                    torch.matmul(p.transpose(2, 3), g)]
        return out


def _run_paged(state):
    case = state["case"]
    scale = 1.0 / math.sqrt(case["d"])
    if own:
        with torch.no_grad():
            return [_framework().paged_attention(state["q"], state["k_pages"], state["v_pages"],
                                                 state["table"], state["lengths"], scale,
                                                 cap=state["cap"], slopes=state["slopes"])]
    b, h, hk, d, page = (case[n] for n in ("b", "h", "hk", "d", "page"))
    table = state["table"].long()
    n = table.shape[1] * page
    k, v = (_cached(state[x][table].permute(0, 2, 1, 3, 4), d).reshape(b, hk, n, d)
            for x in ("k_pages", "v_pages"))
    q = state["q"].float().view(b, hk, h // hk, d)
    x = torch.matmul(q, k.transpose(2, 3)) * scale
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    j = torch.arange(n, device=DEVICE)
    if state["slopes"] is not None:
        far = (state["lengths"][:, None] - 1 - j).float()
        x = x - state["slopes"].view(hk, h // hk, 1) * far[:, None, None, :]
    p = _softmax(x, j < state["lengths"][:, None, None, None])
    return [torch.matmul(p, v).view(b, h, 1, d).to(state["q"].dtype)]


def _run_append(state):
    case = state["case"]
    s, page, d, dtype = case["s"], case["page"], case["d"], state["q"].dtype
    if own:
        cfa = _framework()
        with torch.no_grad():
            q = cfa.paged_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                                 state["table"], state["lengths"], counts=state["counts"], q=state["q"],
                                 frequencies=state["frequencies"], interleaved=case["interleaved"])
            k, v = cfa.paged_read(state["k_pages"], state["v_pages"], state["table"], state["after"], s,
                                  starts=state["lengths"], dtype=dtype)
        return [q, k, v, state["k_pages"], state["v_pages"]]
    i = torch.arange(s, device=DEVICE)
    at = state["lengths"].long()[:, None] + i
    angle = at[:, None, :, None].double() * state["frequencies"]
    cos, sin = torch.cos(angle), torch.sin(angle)
    q = _rotate(state["q"], cos.float(), sin.float(), case["interleaved"])
    # (The 4-bit codes of the keys: of values in 64 bits, since a code is next to a border.)
    k = _rotate(state["k"], cos, sin, case["interleaved"])
    put = at < state["after"][:, None]
    row = torch.arange(case["b"], device=DEVICE)[:, None].expand_as(at)[put]
    pages, slots = state["table"].long()[row, at[put] // page], at[put] % page
    out = [q.to(dtype)]
    for name, x in (("k_pages", k), ("v_pages", state["v"].float())):
        rows = _encode(x.transpose(1, 2)[put])
        state[name][pages, :, slots] = rows
        back = torch.zeros(case["b"], s, case["hk"], d, dtype=dtype, device=DEVICE)
        back[put] = _decode(rows, d).to(dtype)
        out.append(back.transpose(1, 2).contiguous())
    return out + [state["k_pages"], state["v_pages"]]


def _run_read(state):
    case = state["case"]
    s, page, dtype = case["s"], case["page"], _TYPES[case["dtype"]]
    if own:
        with torch.no_grad():
            return list(_framework().paged_read(state["k_pages"], state["v_pages"], state["table"],
                                                state["lengths"], s, starts=state["starts"], dtype=dtype))
    at = state["starts"].long()[:, None] + torch.arange(s, device=DEVICE)
    have = at < state["lengths"][:, None]
    at = at.minimum(torch.full_like(at, state["table"].shape[1] * page - 1))
    pages, slots = state["table"].long().gather(1, at // page), at % page
    return [(_cached(state[x][pages, :, slots], case["d"]) * have[..., None, None]).to(dtype)
            .transpose(1, 2).contiguous() for x in ("k_pages", "v_pages")]


def run(state):
    return {"scored": _run_scored, "paged": _run_paged, "append": _run_append,
            "read": _run_read}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------


def _cache_bytes(case, cache):
    """Of one head's row: what its values take, their scales among them, without padding."""
    d = case["d"]
    return d // 2 + d // 32 if cache == "fp4" else d * _SIZE[cache]


def work(case):
    """Every input read once, every output written once; 4 d operations for a visible query and key
    forward, 10 d backward, three for a rotated value, one for a value converted."""
    op, b, d, hk = case["op"], case["b"], case["d"], case["hk"]
    if op == "scored":
        q, kv = b * case["sq"] * case["h"] * d, b * case["sk"] * hk * d
        moved = 2 * q + 2 * kv + (b * case["sk"] if _masked(case) else 0)
        if case["train"]:  # again q, O, dO, k, v; dQ, dK, dV
            moved += 4 * q + 4 * kv
        return {"bytes": 4 * moved,
                "flops": max(1, (14 if case["train"] else 4) * d * case["h"] * _pairs(case))}
    if op == "paged":
        total = sum(_held(case))
        return {"bytes": 2 * total * hk * _cache_bytes(case, case["cache"])
                + 2 * b * case["h"] * d * _SIZE[case["dtype"]],
                "flops": max(1, 4 * total * case["h"] * d)}
    if op == "append":
        tokens, new, size = b * case["s"], sum(_counts(case)), _SIZE[case["dtype"]]
        rows = 2 * new * hk * _cache_bytes(case, "fp4")
        # (Written, and read back.)
        return {"bytes": 2 * tokens * case["h"] * d * size + 2 * new * hk * d * size + 2 * rows
                + 2 * tokens * hk * d * size + 16 * b,
                "flops": 3 * (tokens * case["h"] + new * hk) * case["dim"] + 4 * new * hk * d}
    got = sum(min(n, case["s"]) for n in _held(case))
    return {"bytes": 2 * hk * (got * _cache_bytes(case, case["cache"])
                               + b * case["s"] * d * _SIZE[case["dtype"]]) + 8 * b,
            "flops": max(1, 2 * got * hk * d)}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------


def _exact_scored(case, seed):
    """Sample by sample and key head by key head; the gradients by torch's differentiation."""
    st = _scored_inputs(case, seed)
    b, h, hk, sq, sk, d = (case[n] for n in ("b", "h", "hk", "sq", "sk", "d"))
    rep, pos = h // hk, torch.arange(sk, device=DEVICE)
    mine = pos[sk - sq:]
    out = [torch.zeros(t.shape, dtype=torch.float64, device=DEVICE)
           for t in (st["q"], st["q"], st["k"], st["v"])]
    for i in range(b):
        hidden = torch.zeros(sq, sk, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden |= pos[None, :] > mine[:, None]
            if st["prefix"] is not None:
                hidden[:, :int(st["prefix"][i])] = False
        if st["documents"] is not None:
            ids = st["documents"][i]
            hidden |= ids[None, :] != ids[mine][:, None]
            hidden |= ids[None, :] < 0
        empty = hidden.all(-1)
        for n in range(hk):
            heads = slice(n * rep, (n + 1) * rep)
            q, k, v = (t.double().detach().requires_grad_(True)
                       for t in (st["q"][i, heads], st["k"][i, n], st["v"][i, n]))
            with torch.enable_grad():
                y = (q.reshape(rep * sq, d) @ k.t()).view(rep, sq, sk) / math.sqrt(d)
                if case["cap"]:
                    y = case["cap"] * torch.tanh(y / case["cap"])
                if case["slopes"]:
                    y = y - st["slopes"][heads, None, None].double() * (mine[:, None] - pos).abs()
                y = y.masked_fill(hidden & ~empty[:, None], -math.inf)
                o = (torch.softmax(y, -1).view(rep * sq, sk) @ v).view(rep, sq, d)
                o = o.masked_fill(empty[:, None], 0.0)
            out[0][i, heads] = o.detach()
            if case["train"]:
                grads = torch.autograd.grad(o, (q, k, v), st["g"][i, heads].double())
                out[1][i, heads], out[2][i, n], out[3][i, n] = grads
    return out if case["train"] else out[:1]


def _values(rows, d):
    """What a cache's rows hold, in 64 bits."""
    if rows.dtype != torch.uint8:
        return rows.double()
    codes = torch.empty(*rows.shape[:-1], d, dtype=torch.long, device=rows.device)
    codes[..., 0::2], codes[..., 1::2] = rows[..., :d // 2] % 16, rows[..., :d // 2] // 16
    code = codes % 8  # (an exponent of two bits, 0 for the subnormal 0.5, and one bit of significand)
    size = torch.where(code < 2, code * 0.5, (1 + (code % 2) * 0.5) * 2.0 ** (code // 2 - 1).double())
    sign = 1.0 - 2.0 * (codes // 8)
    e = rows[..., d // 2:d // 2 + d // 32].double() - 127
    return sign * size * torch.exp2(e).repeat_interleave(32, dim=-1)


def _nearest(x):
    """x [..., d] in 64 bits as the 4-bit values nearest to it."""
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=DEVICE)
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True).clamp_min(1e-300)
    unit = torch.exp2(torch.ceil(torch.log2(top / 7.0)))
    unit = torch.where(top <= 3.5 * unit, unit / 2, torch.where(top > 7 * unit, unit * 2, unit))
    u = (g / unit).abs()
    low = (torch.searchsorted(levels, u.contiguous(), right=True) - 1).clamp_max(6)
    below, above = u - levels[low], levels[low + 1] - u
    up = (above < below) | ((above == below) & (low % 2 == 1))
    return (levels[low + up] * unit * torch.sign(g)).flatten(-2)


def _exact_paged(case, seed):
    st = _paged_inputs(case, seed)
    b, h, hk, d = (case[n] for n in ("b", "h", "hk", "d"))
    out = torch.zeros(b, h, 1, d, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(_held(case)):
        if n == 0:
            continue
        used = st["table"][i, :-(-n // case["page"])].long()
        k, v = (_values(st[x][used].transpose(0, 1).flatten(1, 2)[:, :n], d)
                for x in ("k_pages", "v_pages"))
        q = st["q"][i, :, 0].double().view(hk, h // hk, d)
        y = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        if case["cap"]:
            y = case["cap"] * torch.tanh(y / case["cap"])
        if case["slopes"]:
            back = torch.arange(n - 1, -1, -1, dtype=torch.float64, device=DEVICE)
            y = y - st["slopes"].double().view(hk, -1, 1) * back
        out[i] = torch.matmul(torch.softmax(y, dim=-1), v).view(h, 1, d)
    return [out]


def _turned(x, positions, frequencies, interleaved):
    """x [h, s, d] in 64 bits as complex pairs times e^(i position frequency)."""
    n = 2 * frequencies.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                       positions.double()[:, None] * frequencies)
    head = x[..., :n].double()
    pairs = head.unflatten(-1, (n // 2, 2)) if interleaved else (
        head.unflatten(-1, (2, n // 2)).transpose(-1, -2))
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., n:].double()), dim=-1)


def _exact_append(case, seed):
    """The turned queries, the new tokens as the cache holds them; the pages' bytes are no numbers."""
    st = _append_inputs(case, seed)
    q, k, v = (torch.zeros(st[n].shape, dtype=torch.float64, device=DEVICE) for n in ("q", "k", "v"))
    for i, (have, new) in enumerate(zip(_held(case), _counts(case))):
        at = torch.arange(have, have + case["s"], device=DEVICE)
        q[i] = _turned(st["q"][i], at, st["frequencies"], case["interleaved"])
        k[i, :, :new] = _nearest(_turned(st["k"][i], at, st["frequencies"], case["interleaved"])[:, :new])
        v[i, :, :new] = _nearest(st["v"][i, :, :new].double())
    return [q, k, v, None, None]


def _exact_read(case, seed):
    st = _read_inputs(case, seed)
    b, hk, s, d = (case[n] for n in ("b", "hk", "s", "d"))
    out = []
    for name in ("k_pages", "v_pages"):
        x = torch.zeros(b, hk, s, d, dtype=torch.float64, device=DEVICE)
        for i, n in enumerate(_held(case)):
            first = max(0, n - s)
            t = torch.arange(first, n, device=DEVICE)
            rows = st[name][st["table"][i].long()[t // case["page"]], :, t % case["page"]]
            x[i, :, :n - first] = _values(rows, d).transpose(0, 1)
        out.append(x)
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"scored": _exact_scored, "paged": _exact_paged, "append": _exact_append,
                "read": _exact_read}[case["op"]](case, seed)
