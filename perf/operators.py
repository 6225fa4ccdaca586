"""The attention block of a batch of sequences with a 4-bit KV cache: head
norms with the rotary rotation, causal attention over packed prompts, the
cache's write and read-back, and decode attention over it.

With own False every operator runs in its plain form, elementary torch
operations in 32 bits (angles in 64); with own True through the framework.
Head counts and sizes are those of the repository's two decoder shapes
(14 query and 2 key/value heads of 64; 28 and 4 of 128) or generic ones.
"""
import math

import numpy as np
import torch

own = False

HEADS = ((14, 2), (28, 4), (16, 2), (8, 8), (40, 8), (5, 1))  # (query, key/value) heads
ROPE_THETA = 1e6
EPS = 1e-6


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of one decode step: latency
        _rope("rope_1_token_h14_d64", 1, 14, 2, 64, start=602),
        # the prompt of the 602-token workload, rows of one fused q/k/v product
        _rope("rope_602_tokens_h14_d64", 602, 14, 2, 64, fused=True),
        # many prompts' tokens at once, late in long contexts
        _rope("rope_16384_tokens_h28_d128", 16384, 28, 4, 128, start=100_000),
        # one prompt, the 602-token workload's layer
        _prompt("prompt_602_h14_d64", 602, 1, 14, 2, 64),
        # a server's mixed prompts, packed, with rows of padding behind them
        _prompt("prompt_33_ragged_h28_d128", 1100, 33, 28, 4, 128, mix=3, tail=37),
        # one long prompt
        _prompt("prompt_8192_h28_d128", 8192, 1, 28, 4, 128),
        # the cache rows of one decode step of 64 sequences
        _write("store_64_tokens_h4_d128", 64, 64, 2048, 4, 128),
        # the cache rows of packed prompts
        _write("store_8191_tokens_h4_d128", 8191, 16, 2048, 4, 128),
        # one sequence with a short history: latency
        _decode("decode_1x96_h14_d64", 1, 96, 14, 2, 64, full=True),
        # one sequence with a long history: its positions split over the machine
        _decode("decode_1x32768_h28_d128", 1, 32768, 28, 4, 128, full=True),
        # the 64-sequence workload, histories of all lengths up to 2048
        _decode("decode_64_ragged_2048_h28_d128", 64, 2048, 28, 4, 128),
        # long contexts served together
        _decode("decode_16x65536_h28_d128", 16, 65536, 28, 4, 128, full=True),
    ]


def _rope(name, tokens, heads, kv, dim, start=0, fused=False, neox=True):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv": kv, "dim": dim,
            "start": start, "fused": fused, "neox": neox}


def _prompt(name, longest, seqs, heads, kv, dim, mix=0, tail=0, fused=False):
    # mix 0: every sequence has `longest` tokens; else lengths spread from it down to 0 or 1
    return {"name": name, "op": "prompt", "longest": longest, "seqs": seqs, "heads": heads,
            "kv": kv, "dim": dim, "mix": mix, "tail": tail, "fused": fused}


def _write(name, tokens, slots, room, kv, dim, layers=1, padding=0):
    return {"name": name, "op": "store", "tokens": tokens, "slots": slots, "room": room, "kv": kv,
            "dim": dim, "layers": layers, "padding": padding}


def _decode(name, columns, room, heads, kv, dim, full=False, mix=1, layers=1):
    # full: every column sees `room` positions; else between none and all of them
    return {"name": name, "op": "decode", "columns": columns, "room": room, "heads": heads,
            "kv": kv, "dim": dim, "full": full, "mix": mix, "layers": layers}


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("rope", "prompt", "store", "decode"))
    heads, kv = rng.choice(HEADS)
    mix = rng.randrange(1, 1000)
    if op == "rope":
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        tokens = _log(rng, 1, min(16384, 60_000_000 // ((heads + kv) * dim)))
        case = _rope("", tokens, heads, kv, dim, start=rng.choice((0, 7, 4096, 1_000_000)),
                     fused=rng.random() < 0.5, neox=rng.random() < 0.7)
    elif op == "prompt":
        dim = rng.choice((32, 64, 80, 96, 128))
        seqs = _log(rng, 1, 64)
        most = int(math.sqrt(28 * 8192 * 8192 * 0.5 / (heads * seqs)))
        case = _prompt("", _log(rng, 1, min(8192, most)), seqs, heads, kv, dim, mix=mix,
                       tail=rng.choice((0, 0, 1, 130)), fused=rng.random() < 0.3)
    elif op == "store":
        dim = rng.choice((32, 64, 96, 128))
        tokens = _log(rng, 1, 8191)
        slots = _log(rng, 1, 64)
        case = _write("", tokens, slots, -(-tokens // slots) + rng.randrange(0, 300), kv, dim,
                      layers=rng.randrange(1, 3), padding=rng.choice((0, 0, 3)) if tokens > 3 else 0)
    else:
        dim = rng.choice((32, 64, 96, 128))
        columns = _log(rng, 1, 64)
        room = _log(rng, 1, min(65536, 300_000_000 // (columns * kv * dim)))
        case = _decode("", columns, room, heads, kv, dim, full=rng.random() < 0.3, mix=mix,
                       layers=rng.randrange(1, 3))
    del case["name"]
    return case


def _lengths(case):
    """Tokens of each sequence of a packed prompt."""
    if not case["mix"]:
        return [case["longest"]] * case["seqs"]
    r = np.random.RandomState(case["mix"])
    n = np.floor(r.uniform(0, 1, case["seqs"]) ** 2 * (case["longest"] + 1)).astype(int)
    n[r.randint(case["seqs"])] = case["longest"]
    return n.tolist()


def _visible(case):
    """Positions that each column of a decode step sees."""
    if case["full"]:
        return [case["room"]] * case["columns"]
    r = np.random.RandomState(case["mix"])
    n = np.floor(r.uniform(0, 1, case["columns"]) * (case["room"] + 1)).astype(int)
    return n.tolist()


def work(case):
    d = case["dim"]
    if case["op"] == "rope":
        values = case["tokens"] * (case["heads"] + case["kv"]) * d
        return {"bytes": 8 * values + 4 * case["tokens"], "flops": 8 * values}
    if case["op"] == "prompt":
        n = _lengths(case)
        pairs = sum(x * (x + 1) // 2 for x in n)
        return {"bytes": 4 * sum(n) * d * (2 * case["heads"] + 2 * case["kv"]),
                "flops": 4 * d * case["heads"] * pairs}
    if case["op"] == "store":
        values = 2 * (case["tokens"] - case["padding"]) * case["kv"] * d
        # in as f32, out in 4 bits with a 16-bit scale for 32 values, and both ways again
        return {"bytes": 2 * (values * 4 + values // 2 + values // 16), "flops": 6 * values}
    n = _visible(case)
    cache = 2 * sum(n) * case["kv"] * (d // 2 + d // 16)
    return {"bytes": cache + 8 * case["columns"] * case["heads"] * d,
            "flops": 4 * d * case["heads"] * sum(n)}


# ------------------------------------------------------------------ inputs
def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _qkv(g, tokens, case):
    """Queries, keys and values, either apart or as the rows of one product."""
    h, kv, d = case["heads"], case["kv"], case["dim"]
    if case["fused"]:
        x = _randn(g, tokens, h + 2 * kv, d)
        return x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    return _randn(g, tokens, h, d), _randn(g, tokens, kv, d), _randn(g, tokens, kv, d)


def _rows(g, n, case):
    """Key and value rows: keys have a few channels that are far larger than the others."""
    k, v = _randn(g, n, case["kv"], case["dim"]), _randn(g, n, case["kv"], case["dim"])
    k[..., :: 24] *= 4.0
    return k, v


def prepare(case, seed):
    g = _rng(seed)
    if case["op"] == "rope":
        q, k, _ = _qkv(g, case["tokens"], case)
        scale = torch.exp(_randn(g, case["tokens"], 1, 1))
        if not case["fused"]:
            q, k = q * scale, k * scale
        pos = torch.randint(case["start"], case["start"] + 2 * case["tokens"], (case["tokens"],),
                            generator=g, device="cuda", dtype=torch.int32)
        return {"case": case, "q": q, "k": k, "positions": pos,
                "qw": 1 + 0.1 * _randn(g, case["dim"]), "kw": 1 + 0.1 * _randn(g, case["dim"])}
    if case["op"] == "prompt":
        n = _lengths(case)
        total = sum(n) + case["tail"]
        q, k, v = _qkv(g, total, case)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")
        return {"case": case, "q": q, "k": k, "v": v, "starts": starts,
                "out": torch.zeros(total, case["heads"], case["dim"], device="cuda")}
    if case["op"] == "store":
        k, v = _rows(g, case["tokens"], case)
        # token i goes to slot i mod slots, at positions in a shuffled order
        i = torch.arange(case["tokens"], device="cuda")
        order = torch.randperm(case["room"], generator=g, device="cuda")
        slots = (i % case["slots"]).to(torch.int32)
        positions = order[i // case["slots"]].to(torch.int32)
        if case["padding"]:
            positions[-case["padding"]:] = -1
        return {"case": case, "k": k, "v": v, "slots": slots, "positions": positions,
                "k_out": torch.zeros_like(k), "v_out": torch.zeros_like(v),
                "cache": _cache(case, case["slots"])}
    slots = case["columns"]
    cache = _cache(case, slots)
    step = max(1, 8192 // slots)
    for p in range(0, case["room"], step):
        m = min(step, case["room"] - p)
        k, v = _rows(g, slots * m, case)
        s = torch.arange(slots, device="cuda", dtype=torch.int32).repeat_interleave(m)
        at = torch.arange(p, p + m, device="cuda", dtype=torch.int32).repeat(slots)
        _store(cache, case["layers"] - 1, k, v, s, at)
    order = torch.randperm(slots, generator=g, device="cuda").to(torch.int32)
    return {"case": case, "q": _randn(g, slots, case["heads"], case["dim"]), "cache": cache,
            "lengths": torch.tensor(_visible(case), dtype=torch.int32, device="cuda"),
            "slots": order}


def _cache(case, slots):
    """The cache that a serving program keeps: the framework's, or codes and scales as tensors."""
    if own:
        return _pkg().KvCacheQ40(case["layers"], slots, case["room"], case["kv"], case["dim"])
    # one row more than the cache has positions: where padding rows go
    shape = (case["layers"], slots, case["kv"], case["room"] + 1)
    zero = torch.zeros
    return {"codes": [zero(*shape, case["dim"] // 2, dtype=torch.uint8, device="cuda") for _ in "kv"],
            "scales": [zero(*shape, case["dim"] // 32, dtype=torch.float16, device="cuda") for _ in "kv"]}


def _store(cache, layer, k, v, slots, positions):
    if own:
        cache.write(layer, k, v, positions, slots)
    else:
        _plain_store(cache, layer, k, v, slots, positions)


# ------------------------------------------------------------------ plain forms
def _plain_norm_rope(x, weight, angle, neox):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    half = x.shape[-1] // 2
    a, b = (y[..., :half], y[..., half:]) if neox else (y[..., 0::2], y[..., 1::2])
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    r, t = a * c - b * s, a * s + b * c
    return torch.cat([r, t], -1) if neox else torch.stack([r, t], -1).flatten(-2)


def _plain_softmax(s):
    """Weights and their sum; a row with nothing visible has weights and sum 0."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return p, p.sum(-1, keepdim=True)


def _plain_prompt(q, k, v, starts, longest, out):
    seqs, total = starts.numel() - 1, q.shape[0]
    h, kv, d = q.shape[1], k.shape[1], q.shape[2]
    n = starts[1:] - starts[:-1]
    at = torch.arange(longest, device=q.device)
    rows = (starts[:-1, None] + at).clamp(max=total - 1).long()
    group = lambda x: x[rows].permute(0, 2, 1, 3)  # noqa: E731
    qs = group(q).reshape(seqs, kv, h // kv, longest, d)
    s = qs @ group(k).transpose(-1, -2)[:, :, None] * (1.0 / math.sqrt(d))
    seen = (at[None, :] <= at[:, None]) & (at[None, None, :] < n[:, None, None])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p, norm = _plain_softmax(s)
    o = (p @ group(v)[:, :, None]) / norm.clamp(min=1e-30)
    o = o.reshape(seqs, h, longest, d)
    token = torch.arange(total, device=q.device, dtype=torch.int32)
    seq = (torch.searchsorted(starts, token, right=True) - 1).clamp(max=seqs - 1)
    place = (token - starts[seq]).clamp(max=longest - 1).long()
    return torch.where((token < starts[-1])[:, None, None], o[seq, :, place], out)


def _half_bits(x):
    """fp16 values of non-negative x by the block format's rounding: halves go up."""
    bits = x.view(torch.int32)
    e = (bits >> 23) - 112
    m = bits & 0x7FFFFF
    low = ((m | 0x800000) >> (1 - e).clamp(0, 31)) + 0x1000 >> 13
    bits = torch.where(e <= 0, torch.where(e < -10, torch.zeros_like(m), low),
                       (e << 10) + (m + 0x1000 >> 13))
    return bits.clamp(max=0x7C00).to(torch.int16).view(torch.float16)


def _plain_quantize(x):
    """Codes (two to a byte: value j of a block low, j + 16 high) and scales of 32-value blocks."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    scale = _half_bits(top / torch.full_like(top, 7.0))
    stored = scale.float()
    inverse = torch.where(stored == 0, torch.zeros_like(stored), torch.ones_like(stored) / stored)
    y = (b * inverse[..., None] + 8.0).clamp(0, 15.5)
    whole = y.floor()
    code = (whole + (y - whole >= 0.5)).clamp(max=15).to(torch.uint8)
    code = torch.where((top > 0)[..., None], code, torch.zeros_like(code))
    return (code[..., :16] | code[..., 16:] << 4).flatten(-2), scale


def _plain_values(codes, scales):
    c = codes.reshape(*codes.shape[:-1], -1, 16)
    return ((torch.cat([c & 15, c >> 4], -1).float() - 8.0) * scales.float()[..., None]).flatten(-2)


def _plain_store(cache, layer, k, v, slots, positions):
    s = slots.long()
    for x, codes, scales in zip((k, v), cache["codes"], cache["scales"]):
        p = torch.where(positions < 0, codes.shape[3] - 1, positions.long())
        codes[layer][s, :, p], scales[layer][s, :, p] = _plain_quantize(x)


def _plain_read(cache, layer, slots, positions, outs):
    s, p = slots.long(), positions.long()
    keep = (p >= 0)[:, None, None]
    p = p.clamp(min=0)
    return [torch.where(keep, _plain_values(c[layer][s, :, p], d[layer][s, :, p]), out)
            for c, d, out in zip(cache["codes"], cache["scales"], outs)]


def _plain_decode(q, cache, layer, slots, lengths):
    columns, h, d = q.shape
    k, v = (_plain_values(c[layer][slots.long()], s[layer][slots.long()])
            for c, s in zip(cache["codes"], cache["scales"]))
    kv, room = k.shape[1], k.shape[2]
    s = q.reshape(columns, kv, h // kv, d) @ k.transpose(-1, -2) * (1.0 / math.sqrt(d))
    seen = torch.arange(room, device=q.device)[None] < lengths[:, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p, norm = _plain_softmax(s)
    return ((p @ v) / norm.clamp(min=1e-30)).reshape(columns, h, d)


def run(state):
    case = state["case"]
    if case["op"] == "rope":
        if own:
            return _pkg().qk_norm_rope(state["q"], state["k"], state["qw"], state["kw"],
                                       state["positions"], ROPE_THETA, EPS, case["neox"])
        i = torch.arange(case["dim"] // 2, device="cuda", dtype=torch.float64)
        angle = state["positions"].double()[:, None] * ROPE_THETA ** (-2.0 * i / case["dim"])
        return (_plain_norm_rope(state["q"], state["qw"], angle, case["neox"]),
                _plain_norm_rope(state["k"], state["kw"], angle, case["neox"]))
    if case["op"] == "prompt":
        if own:
            return _pkg().attention_prompt(state["q"], state["k"], state["v"], state["starts"],
                                           out=state["out"])
        return _plain_prompt(state["q"], state["k"], state["v"], state["starts"], case["longest"],
                             state["out"])
    layer = case["layers"] - 1
    if case["op"] == "store":
        _store(state["cache"], layer, state["k"], state["v"], state["slots"], state["positions"])
        if own:
            return state["cache"].read(layer, state["positions"], state["slots"],
                                       k_out=state["k_out"], v_out=state["v_out"])
        return _plain_read(state["cache"], layer, state["slots"], state["positions"],
                           (state["k_out"], state["v_out"]))
    if own:
        return state["cache"].attention(state["q"], layer, state["lengths"], state["slots"])
    return _plain_decode(state["q"], state["cache"], layer, state["slots"], state["lengths"])


# ------------------------------------------------------------------ 64 bits
def _exact_softmax_sum(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the visible keys, rows of q, all in 64 bits."""
    s = torch.einsum("id,jd->ij", q, k) / math.sqrt(q.shape[-1])
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, -1)
    return torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p)) @ v


def _exact_block_values(x):
    """The values that 4-bit blocks hold, step by step in the format's own roundings."""
    x = x.double().cpu().numpy()
    b = x.reshape(-1, 32)
    f32 = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    top = np.abs(b).max(-1, keepdims=True)
    want = f32(top / 7.0)
    # steps of fp16: 11 significant bits, none finer than 2^-24; halves away from zero
    with np.errstate(divide="ignore"):
        e = np.where(want > 0, np.floor(np.log2(np.where(want > 0, want, 1.0))), 0.0)
    step = 2.0 ** np.maximum(e - 10, -24)
    d = np.floor(want / step + 0.5) * step
    inverse = np.divide(1.0, d, out=np.zeros_like(d), where=d > 0)
    y = f32(f32(b * f32(inverse)) + 8.0)
    n = np.clip(np.trunc(y + np.copysign(0.5, y)), 0, 15)
    return np.where(top > 0, f32(d * (n - 8.0)), 0.0).reshape(x.shape)


def exact(case, seed):
    global own
    if case["op"] == "prompt" and sum(n * n for n in _lengths(case)) * case["heads"] > 2_000_000_000:
        return None
    if case["op"] == "decode" and sum(_visible(case)) * case["kv"] * case["dim"] > 600_000_000:
        return None
    was, own = own, False  # the inputs, apart from the framework
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rope":
        outs = []
        d = case["dim"]
        pos = state["positions"].double()
        for x, w in ((state["q"], state["qw"]), (state["k"], state["kw"])):
            x = x.double()
            n = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
            out = torch.empty_like(n)
            for i in range(d // 2):
                phase = pos * math.pow(ROPE_THETA, -2.0 * i / d)
                c, s = torch.cos(phase)[:, None], torch.sin(phase)[:, None]
                lo, hi = (i, i + d // 2) if case["neox"] else (2 * i, 2 * i + 1)
                out[..., lo] = n[..., lo] * c - n[..., hi] * s
                out[..., hi] = n[..., hi] * c + n[..., lo] * s
            outs.append(out)
        return tuple(outs)
    if case["op"] == "prompt":
        q, k, v = (state[x].double() for x in "qkv")
        out = state["out"].double()
        a, group = 0, case["heads"] // case["kv"]
        for n in _lengths(case):
            seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            for h in range(case["heads"] if n else 0):
                out[a:a + n, h] = _exact_softmax_sum(q[a:a + n, h], k[a:a + n, h // group],
                                                     v[a:a + n, h // group], seen)
            a += n
        return out
    if case["op"] == "store":
        outs = []
        for x in (state["k"], state["v"]):
            y = _exact_block_values(x)
            y[state["positions"].cpu().numpy() < 0] = 0.0
            outs.append(y)
        return outs
    layer, group = case["layers"] - 1, case["heads"] // case["kv"]
    q = state["q"].double()
    out = torch.zeros_like(q)
    for c, n in enumerate(_visible(case)):
        slot = int(state["slots"][c])
        for h in range(case["kv"] if n else 0):
            k, v = ((torch.stack([x[layer][slot, h, :n].view(n, -1, 16) & 15,
                                  x[layer][slot, h, :n].view(n, -1, 16) >> 4], 2).double() - 8)
                    .view(n, -1, 32) * s[layer][slot, h, :n].double()[..., None]
                    for x, s in zip(state["cache"]["codes"], state["cache"]["scales"]))
            rows = slice(h * group, (h + 1) * group)
            out[c, rows] = _exact_softmax_sum(q[c, rows], k.reshape(n, -1), v.reshape(n, -1),
                                              torch.ones(group, n, dtype=torch.bool, device="cuda"))
    return out
