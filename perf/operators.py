"""Timed workloads of the operators around self-attention, called as a user's program calls them:
rotary positions, the append to a paged key-value cache, the attention of one new token over that
cache, and cross attention to states of another length.

A case is one call pattern. `op` names the operator:
  rotary      fused_rotary on q [b, h, s, d] and k [b, hk, s, d] (views of [b, s, heads, d] buffers),
              or, with "qkv", fused_rotary_qkv on one [b, s, 3 h d] projection; with "train" the
              backward too;
  append      paged_append of `s` new tokens (ragged with "ragged") to caches that hold lo .. hi
              tokens, keys and queries rotated on the way;
  paged       paged_attention of one token per sequence over lo .. hi cached tokens;
  cross       fused_cross_attention of sq queries to sk keys, of which each sample sees lo .. sk
              ("lo" absent: all); with "train" the backward too.
Inputs are N(0, 1), scale 1 / sqrt(d). Types: `dtype` is the activations', `cache` the cache's.

With `own` false the same results come from elementary torch operations in 32 bits (angles in 64).
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
_PKG = str(Path(__file__).resolve().parent.parent / "candle-fused-attn_amd")
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import candle_fused_attn
    return candle_fused_attn


def listed():
    return [
        # The positions of one new token for each of a few sequences: launch latency.
        {"name": "rotary_token", "op": "rotary", "b": 8, "h": 6, "hk": 6, "s": 1, "d": 64, "dim": 64,
         "dtype": "f32", "interleaved": False, "factor": 1.0, "far": 4096, "qkv": False,
         "train": False},
        # A training step's rotation of a fused projection, at the benchmark's shape.
        {"name": "rotary_train", "op": "rotary", "b": 64, "h": 6, "hk": 6, "s": 240, "d": 64,
         "dim": 64, "dtype": "f32", "interleaved": False, "factor": 1.0, "far": 0, "qkv": True,
         "train": True},
        # A long chunk of a long context: half of each head rotated, pairs interleaved, stretched
        # frequencies, grouped key heads, positions past a hundred thousand, an odd length.
        {"name": "rotary_long", "op": "rotary", "b": 2, "h": 32, "hk": 8, "s": 8191, "d": 128,
         "dim": 64, "dtype": "bf16", "interleaved": True, "factor": 8.0, "far": 120000, "qkv": False,
         "train": False},
        # One decoding step of a batch: one token each into caches of any fill.
        {"name": "append_token", "op": "append", "b": 64, "h": 6, "hk": 6, "s": 1, "d": 64, "dim": 64,
         "dtype": "f32", "cache": "f32", "page": 16, "lo": 1, "hi": 1000, "interleaved": False,
         "ragged": False},
        # The prompts of a batch, padded to the longest, into empty caches.
        {"name": "append_prompts", "op": "append", "b": 16, "h": 32, "hk": 8, "s": 2048, "d": 128,
         "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 64, "lo": 0, "hi": 0,
         "interleaved": False, "ragged": True},
        # A chunk of fp32 activations behind what half-precision caches hold already, narrow heads.
        {"name": "append_chunk", "op": "append", "b": 5, "h": 12, "hk": 12, "s": 333, "d": 32,
         "dim": 32, "dtype": "f32", "cache": "f16", "page": 32, "lo": 0, "hi": 700,
         "interleaved": True, "ragged": True},
        # One short sequence, one small layer: latency.
        {"name": "paged_one", "op": "paged", "b": 1, "h": 6, "hk": 6, "d": 64, "dtype": "f32",
         "cache": "f32", "page": 16, "lo": 240, "hi": 240},
        # A serving batch of unequal sequences, fp32 throughout.
        {"name": "paged_batch", "op": "paged", "b": 64, "h": 6, "hk": 6, "d": 64, "dtype": "f32",
         "cache": "f32", "page": 16, "lo": 1, "hi": 2048},
        # Few very long contexts, grouped wide heads, bf16.
        {"name": "paged_long", "op": "paged", "b": 4, "h": 32, "hk": 8, "d": 128, "dtype": "bf16",
         "cache": "bf16", "page": 64, "lo": 60000, "hi": 131071},
        # One decoding step's query to an encoder's states.
        {"name": "cross_token", "op": "cross", "b": 8, "h": 6, "hk": 6, "sq": 1, "sk": 1536, "d": 64,
         "train": False},
        # A training step of a decoder of the benchmark's shape on padded states of another length.
        {"name": "cross_train", "op": "cross", "b": 64, "h": 6, "hk": 6, "sq": 240, "sk": 1024,
         "d": 64, "lo": 300, "train": True},
        # Wide heads in groups, odd lengths both ways.
        {"name": "cross_grouped_train", "op": "cross", "b": 4, "h": 16, "hk": 4, "sq": 777,
         "sk": 2049, "d": 128, "train": True},
    ]


_MOST = None


def _most():
    """The most bytes and operations a drawn case may cost, by operator: the largest listed one's."""
    global _MOST
    if _MOST is None:
        _MOST = {}
        for case in listed():
            w = work(case)
            for key in ("bytes", "flops"):
                at = (case["op"], key)
                _MOST[at] = max(_MOST.get(at, 0), w[key])
    return _MOST


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hk = rng.choice((1, 2, 3, 4, 6, 8))
    return hk * rng.choice((1, 1, 2, 3, 4, 8)), hk


def _draw(rng):
    op = rng.choice(("rotary", "append", "paged", "cross"))
    h, hk = _heads(rng)
    d = rng.choice((32, 64, 64, 128))
    dtype, cache = rng.choice((("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                               ("bf16", "bf16")))
    if op == "rotary":
        qkv = rng.random() < 0.4
        return {"op": op, "b": _log(rng, 1, 64), "h": h, "hk": h if qkv else hk,
                "s": _log(rng, 1, 8191), "d": d, "dim": rng.choice((d, d, d // 2, d // 4)),
                "dtype": dtype, "interleaved": rng.random() < 0.5,
                "factor": rng.choice((1.0, 4.0, 8.0)), "far": rng.choice((0, 0, 4096, 120000)),
                "qkv": qkv, "train": rng.random() < 0.5}
    if op == "append":
        s = rng.choice((1, _log(rng, 2, 2048)))
        hi = rng.choice((0, _log(rng, 1, 4096)))
        return {"op": op, "b": _log(rng, 1, 64), "h": h, "hk": hk, "s": s, "d": d,
                "dim": rng.choice((d, d, d // 2)), "dtype": dtype, "cache": cache,
                "page": rng.choice((16, 32, 48, 64, 128)), "lo": 0, "hi": hi,
                "interleaved": rng.random() < 0.5, "ragged": s > 1 and rng.random() < 0.7}
    if op == "paged":
        hi = _log(rng, 1, 131071)
        return {"op": op, "b": _log(rng, 1, 128), "h": h, "hk": hk, "d": d, "dtype": dtype,
                "cache": cache, "page": rng.choice((16, 32, 48, 64, 128)),
                "lo": rng.choice((0, 1, hi // 2, hi)), "hi": hi}
    sk = _log(rng, 1, 4096)
    case = {"op": op, "b": _log(rng, 1, 64), "h": h, "hk": hk,
            "sq": rng.choice((1, _log(rng, 1, 16), _log(rng, 16, 2048))), "sk": sk, "d": d,
            "train": rng.random() < 0.5}
    if rng.random() < 0.5:
        case["lo"] = rng.choice((0, 1, sk // 2))
    return case


def draw(rng):
    while True:
        case = _draw(rng)
        w, most = work(case), _most()
        if all(w[key] <= most[case["op"], key] for key in ("bytes", "flops")):
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
    """Tokens each sequence's cache holds before an append, or has for an attention."""
    return _lengths(case["b"], case["lo"], case["hi"])


def _frequencies(dim, factor):
    """Radians per position of each of a head's dim / 2 pairs, 10000^(-2 i / dim); with a factor,
    the slow ones (fewer than one turn over 4096 positions) slowed by it, the fast ones (more than
    32 turns) as they are, a straight line between."""
    f = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * (keep + (1.0 - keep) / factor)).to(DEVICE)


def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(_TYPES[dtype])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


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
    return _normal(gen, case["cache"], *shape), _normal(gen, case["cache"], *shape), rows


def _rotary_inputs(case, seed):
    gen, b, s, d = _generator(seed), case["b"], case["s"], case["d"]
    start = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device=DEVICE)
    st = {"positions": start + torch.arange(s, device=DEVICE)[None, :],
          "frequencies": _frequencies(case["dim"], case["factor"])}
    if case["qkv"]:
        st["x"] = [_normal(gen, case["dtype"], b, s, 3 * case["h"] * d)]
        st["g"] = [_normal(gen, case["dtype"], b, s, 3 * case["h"] * d)]
    else:
        st["x"] = [_normal(gen, case["dtype"], b, s, n, d).transpose(1, 2)
                   for n in (case["h"], case["hk"])]
        st["g"] = [_normal(gen, case["dtype"], b, s, n, d).transpose(1, 2)
                   for n in (case["h"], case["hk"])]
    if not case["train"]:
        del st["g"]
    return st


def _append_inputs(case, seed):
    gen, b, s, d = _generator(seed), case["b"], case["s"], case["d"]
    held, counts = _held(case), _counts(case)
    total = [x + y for x, y in zip(held, counts)]
    kp, vp, table = _pages(gen, case, total, max(total))
    q, k, v = (_normal(gen, case["dtype"], b, s, n, d).transpose(1, 2)
               for n in (case["h"], case["hk"], case["hk"]))
    return {"q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, "table": table,
            "lengths": _ints(held), "counts": _ints(counts) if case["ragged"] else None,
            "frequencies": _frequencies(case["dim"], 1.0)}


def _paged_inputs(case, seed):
    gen, lengths = _generator(seed), _held(case)
    kp, vp, table = _pages(gen, case, lengths, max(lengths))
    return {"q": _normal(gen, case["dtype"], case["b"], case["h"], 1, case["d"]), "k_pages": kp,
            "v_pages": vp, "table": table, "lengths": _ints(lengths)}


def _cross_inputs(case, seed):
    gen, b, d = _generator(seed), case["b"], case["d"]
    q, g = (_normal(gen, "f32", b, case["sq"], case["h"], d).transpose(1, 2) for _ in range(2))
    k, v = (_normal(gen, "f32", b, case["sk"], case["hk"], d).transpose(1, 2) for _ in range(2))
    lengths = _ints(_lengths(b, case["lo"], case["sk"])) if "lo" in case else None
    return {"q": q, "k": k, "v": v, "g": g if case["train"] else None, "lengths": lengths}


_INPUTS = {"rotary": _rotary_inputs, "append": _append_inputs, "paged": _paged_inputs,
           "cross": _cross_inputs}


def prepare(case, seed):
    state = _INPUTS[case["op"]](case, seed)
    if case.get("train"):
        for t in state["x"] if case["op"] == "rotary" else [state["q"], state["k"], state["v"]]:
            t.requires_grad_(True)
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def _angles(positions, frequencies):
    a = positions.double()[..., None] * frequencies
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, interleaved):
    """x [b, h, s, d] rotated by angles [b, 1, s, dim / 2], in 32 bits."""
    x, n = x.float(), cos.shape[-1]
    if interleaved:
        a, c = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * cos - c * sin, c * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, c = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * cos - c * sin, c * cos + a * sin), dim=-1)
    return torch.cat((y, x[..., 2 * n:]), dim=-1)


def _rotary_pass(state, x, sign):
    case = state["case"]
    cos, sin = _angles(state["positions"][:, None], state["frequencies"])
    sin = sin * sign
    if case["qkv"]:
        b, s, w = x[0].shape
        q, k, v = (t.transpose(1, 2) for t in x[0].view(b, s, 3, case["h"], case["d"]).unbind(2))
        parts = [_rotate(q, cos, sin, case["interleaved"]), _rotate(k, cos, sin, case["interleaved"]),
                 v.float()]
        return [torch.stack([t.transpose(1, 2) for t in parts], dim=2).view(b, s, w).to(x[0].dtype)]
    return [_rotate(t, cos, sin, case["interleaved"]).to(t.dtype) for t in x]


def _run_rotary(state):
    case = state["case"]
    if own:
        cfa = _framework()

        def forward():
            if case["qkv"]:
                return [cfa.fused_rotary_qkv(state["x"][0], case["h"], state["positions"],
                                             state["frequencies"], case["interleaved"])]
            return list(cfa.fused_rotary(*state["x"], state["positions"], state["frequencies"],
                                         case["interleaved"]))

        if not case["train"]:
            with torch.no_grad():
                return forward()
        out = forward()
        return [*(t.detach() for t in out), *torch.autograd.grad(out, state["x"], state["g"])]
    with torch.no_grad():
        out = _rotary_pass(state, state["x"], 1.0)
        return out + _rotary_pass(state, state["g"], -1.0) if case["train"] else out


def _run_append(state):
    case = state["case"]
    if own:
        q = _framework().paged_append(
            state["k"], state["v"], state["k_pages"], state["v_pages"], state["table"],
            state["lengths"], counts=state["counts"], q=state["q"],
            frequencies=state["frequencies"], interleaved=case["interleaved"])
        return [q, state["k_pages"], state["v_pages"]]
    s, page = case["s"], case["page"]
    i = torch.arange(s, device=DEVICE)
    at = state["lengths"].long()[:, None] + i
    cos, sin = _angles(at[:, None], state["frequencies"])
    q, k = (_rotate(state[n], cos, sin, case["interleaved"]) for n in ("q", "k"))
    put = torch.ones_like(at, dtype=torch.bool) if state["counts"] is None else (
        i < state["counts"][:, None])
    row = torch.arange(case["b"], device=DEVICE)[:, None].expand_as(at)[put]
    pages, slots = state["table"].long()[row, at[put] // page], at[put] % page
    for name, x in (("k_pages", k), ("v_pages", state["v"])):
        state[name][pages, :, slots] = x.transpose(1, 2)[put].to(state[name].dtype)
    return [q.to(state["q"].dtype), state["k_pages"], state["v_pages"]]


def _softmax(scores, mask):
    """Softmax over the last dimension where `mask` holds; rows that it leaves empty are 0."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _run_paged(state):
    case = state["case"]
    scale = 1.0 / math.sqrt(case["d"])
    if own:
        with torch.no_grad():
            return [_framework().paged_attention(state["q"], state["k_pages"], state["v_pages"],
                                                 state["table"], state["lengths"], scale)]
    b, h, hk, d, page = (case[n] for n in ("b", "h", "hk", "d", "page"))
    table = state["table"].long()
    n = table.shape[1] * page
    k, v = (state[x][table].permute(0, 2, 1, 3, 4).float().reshape(b, hk, n, d)
            for x in ("k_pages", "v_pages"))
    q = state["q"].float().view(b, hk, h // hk, d)
    mask = torch.arange(n, device=DEVICE) < state["lengths"][:, None, None, None]
    p = _softmax(torch.matmul(q, k.transpose(2, 3)) * scale, mask)
    return [torch.matmul(p, v).view(b, h, 1, d).to(state["q"].dtype)]


def _run_cross(state):
    case = state["case"]
    scale = 1.0 / math.sqrt(case["d"])
    leaves = [state["q"], state["k"], state["v"]]
    if own:
        cfa = _framework()
        if not case["train"]:
            with torch.no_grad():
                return [cfa.fused_cross_attention(*leaves, scale, state["lengths"])]
        out = cfa.fused_cross_attention(*leaves, scale, state["lengths"])
        return [out.detach(), *torch.autograd.grad(out, leaves, state["g"])]
    with torch.no_grad():
        b, h, hk, sq, sk, d = (case[n] for n in ("b", "h", "hk", "sq", "sk", "d"))
        q = leaves[0].reshape(b, hk, h // hk * sq, d)
        k, v = (t.contiguous() for t in leaves[1:])
        p = torch.matmul(q, k.transpose(2, 3)) * scale
        mask = torch.ones(1, 1, 1, sk, dtype=torch.bool, device=DEVICE)
        if state["lengths"] is not None:
            mask = torch.arange(sk, device=DEVICE) < state["lengths"][:, None, None, None]
        p = _softmax(p, mask)
        o = torch.matmul(p, v)
        out = [o.view(b, h, sq, d)]
        if case["train"]:
            g = state["g"].reshape(b, hk, h // hk * sq, d)
            ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * o).sum(-1, keepdim=True)) * scale
            out += [torch.matmul(ds, k).view(b, h, sq, d), torch.matmul(ds.transpose(2, 3), q),
                    torch.matmul(p.transpose(2, 3), g)]
        return out


def run(state):
    return {"rotary": _run_rotary, "append": _run_append, "paged": _run_paged,
            "cross": _run_cross}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------


def work(case):
    """Every input read once, every output written once; three operations for a rotated value, 4 d
    for a query and key forward, 10 d backward."""
    op, b, d = case["op"], case["b"], case["d"]
    if op == "rotary":
        tokens, size = b * case["s"], _SIZE[case["dtype"]]
        heads = case["h"] + case["hk"]
        passes = 2 if case["train"] else 1
        moved = tokens * (heads + (case["h"] if case["qkv"] else 0)) * d * size * 2
        return {"bytes": passes * moved + 8 * tokens + 4 * case["dim"],
                "flops": passes * 3 * tokens * heads * case["dim"]}
    if op == "append":
        tokens, new, size = b * case["s"], sum(_counts(case)), _SIZE[case["dtype"]]
        kv = 2 * new * case["hk"] * d * (size + _SIZE[case["cache"]])
        return {"bytes": 2 * tokens * case["h"] * d * size + kv + 12 * b,
                "flops": 3 * (tokens * case["h"] + new * case["hk"]) * case["dim"]}
    if op == "paged":
        total = sum(_held(case))
        return {"bytes": 2 * total * case["hk"] * d * _SIZE[case["cache"]]
                + 2 * b * case["h"] * d * _SIZE[case["dtype"]],
                "flops": max(1, 4 * total * case["h"] * d)}
    keys = sum(_lengths(b, case["lo"], case["sk"])) if "lo" in case else b * case["sk"]
    q, kv = b * case["sq"] * case["h"] * d, keys * case["hk"] * d
    moved = 2 * q + 2 * kv
    if case["train"]:  # again q, O, dO, k, v; dQ, and all of dK and dV
        moved += 4 * q + 2 * kv + 2 * b * case["sk"] * case["hk"] * d
    return {"bytes": 4 * moved,
            "flops": max(1, (14 if case["train"] else 4) * d * case["h"] * case["sq"] * keys)}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------


def _turned(x, positions, frequencies, interleaved, sign=1.0):
    """x [b, h, s, d] in 64 bits as complex pairs times e^(i position frequency)."""
    n = 2 * frequencies.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                       sign * positions.double()[:, None, :, None] * frequencies)
    head = x[..., :n].double()
    pairs = head.unflatten(-1, (n // 2, 2)) if interleaved else (
        head.unflatten(-1, (2, n // 2)).transpose(-1, -2))
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., n:].double()), dim=-1)


def _exact_rotary(case, seed):
    st = _rotary_inputs(case, seed)

    def turn(tensors, sign):
        if not case["qkv"]:
            return [_turned(t, st["positions"], st["frequencies"], case["interleaved"], sign)
                    for t in tensors]
        b, s, w = tensors[0].shape
        x = tensors[0].view(b, s, 3, case["h"], case["d"])
        y = x.double()
        for i in range(2):
            y[:, :, i] = _turned(x[:, :, i].transpose(1, 2), st["positions"], st["frequencies"],
                                 case["interleaved"], sign).transpose(1, 2)
        return [y.view(b, s, w)]

    return turn(st["x"], 1.0) + (turn(st["g"], -1.0) if case["train"] else [])


def _exact_append(case, seed):
    st = _append_inputs(case, seed)
    held, counts, page = _held(case), _counts(case), case["page"]
    at = st["lengths"].long()[:, None] + torch.arange(case["s"], device=DEVICE)
    q, k = (_turned(st[n], at, st["frequencies"], case["interleaved"]) for n in ("q", "k"))
    kp, vp = st["k_pages"].double(), st["v_pages"].double()
    for i, (have, new) in enumerate(zip(held, counts)):
        t = torch.arange(have, have + new, device=DEVICE)
        where = st["table"][i].long()[t // page], slice(None), t % page
        kp[where] = k[i, :, :new].transpose(0, 1)
        vp[where] = st["v"][i, :, :new].transpose(0, 1).double()
    return [q, kp, vp]


def _exact_paged(case, seed):
    st = _paged_inputs(case, seed)
    b, h, hk, d = (case[n] for n in ("b", "h", "hk", "d"))
    out = torch.zeros(b, h, 1, d, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(_held(case)):
        if n == 0:
            continue
        used = st["table"][i, :-(-n // case["page"])].long()
        k, v = (st[x][used].transpose(0, 1).reshape(hk, -1, d)[:, :n].double()
                for x in ("k_pages", "v_pages"))
        q = st["q"][i, :, 0].double().view(hk, h // hk, d)
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), dim=-1)
        out[i] = torch.matmul(p, v).view(h, 1, d)
    return [out]


def _exact_cross(case, seed):
    st = _cross_inputs(case, seed)
    b, h, hk, sk, d = (case[n] for n in ("b", "h", "hk", "sk", "d"))
    lengths = _lengths(b, case["lo"], sk) if "lo" in case else [sk] * b
    scale, rep = 1.0 / math.sqrt(d), h // hk
    o, dq = (torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
    dk, dv = (torch.zeros(st["k"].shape, dtype=torch.float64, device=DEVICE) for _ in range(2))
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        q = st["q"][i].double()
        k, v = (st[x][i, :, :n].double().repeat_interleave(rep, 0) for x in ("k", "v"))
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * scale, dim=-1)
        o[i] = torch.matmul(p, v)
        if not case["train"]:
            continue
        g = st["g"][i].double()
        ds = torch.matmul(g, v.transpose(1, 2).contiguous()) - (g * o[i]).sum(-1, keepdim=True)
        ds = ds * p * scale
        dq[i] = torch.matmul(ds, k)
        dk[i, :, :n] = torch.matmul(ds.transpose(1, 2).contiguous(), q).view(hk, rep, n, d).sum(1)
        dv[i, :, :n] = torch.matmul(p.transpose(1, 2).contiguous(), g).view(hk, rep, n, d).sum(1)
    return [o, dq, dk, dv] if case["train"] else [o]


def exact(case, seed):
    with torch.no_grad():
        return {"rotary": _exact_rotary, "append": _exact_append, "paged": _exact_paged,
                "cross": _exact_cross}[case["op"]](case, seed)
