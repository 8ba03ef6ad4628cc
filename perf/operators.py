"""Rotary positions, the 8-bit key/value cache, the attention that reads it and the eviction from it: the calls of a
server with long contexts, each in a plain form (elementary torch operations) and as kriya_q4 offers it.

The 8-bit cache holds, for every sequence and key/value head, blocks of 32 tokens: one byte an element (int8 or e4m3)
and one f32 scale a block, with the raw bf16 rows of the last block beside them. Within a block the bytes stand in the
order of the matrix instructions' operands: keys as [head_dim / 16][32 tokens][16], values as
[head_dim / 32][2 h][32 dims][2 a][2 s][4 j] with token 16 s + 8 a + 4 h + j.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
THETA = 1e6
HALF, INTERLEAVED = "half", "interleaved"
LARGEST_FLOPS = 6e10  # of a drawn case; the largest listed one has more
LARGEST_BYTES = 2.5e8
LARGEST_SCORES = 2.4e8  # scores of the plain attention held at once, in elements


def listed():
    return [
        # One decoded token of 16 sequences: q and k, side by side in the row of a fused projection, rotated in place.
        {"name": "rope_b16", "kind": "rope", "tokens": 16, "heads": 18, "row": 20, "head_dim": 128, "rotary": 128,
         "layout": HALF, "dtype": "bf16", "inverse": False, "table": "given", "far": 8192},
        # A prompt whose length stretches the trained context: its table by parts, then a quarter of each head rotated.
        {"name": "rope_m3907", "kind": "rope", "tokens": 3907, "heads": 16, "row": 16, "head_dim": 128, "rotary": 32,
         "layout": INTERLEAVED, "dtype": "f32", "inverse": False, "table": "parts", "far": 131072},
        # The new token of 16 sequences: rotated, quantised into the cache; q rotated beside it.
        {"name": "append_b16", "kind": "append", "batch": 16, "tokens": 16, "past": 511, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8", "rope": True},
        # The prompts of five sequences in one ragged batch, one of them already half in the cache, one empty.
        {"name": "append_m3907", "kind": "append", "batch": 5, "tokens": 3907, "past": 1000, "kv_heads": 8, "q_heads": 0,
         "head_dim": 64, "format": "e4m3", "rope": False},
        # One decoded token of five sequences of different lengths up to 3000: the smallest attention call.
        {"name": "attn_b5", "kind": "attn", "batch": 5, "tokens": 5, "past": 2999, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8"},
        # A large decode batch: 48 sequences up to 8000 positions, few heads to share each row.
        {"name": "attn_b48", "kind": "attn", "batch": 48, "tokens": 48, "past": 7999, "kv_heads": 8, "q_heads": 32,
         "head_dim": 64, "format": "e4m3"},
        # One sequence with a very long context.
        {"name": "attn_b1_long", "kind": "attn", "batch": 1, "tokens": 1, "past": 131071, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8"},
        # A whole prompt, causal: 3907 tokens, a ragged last tile.
        {"name": "attn_m3907", "kind": "attn", "batch": 1, "tokens": 3907, "past": 0, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8"},
        # A step that mixes chunks of prompts with decoded tokens (one sequence has a single new token, one has none).
        {"name": "attn_chunk", "kind": "attn", "batch": 4, "tokens": 600, "past": 12000, "kv_heads": 2, "q_heads": 10,
         "head_dim": 256, "format": "e4m3"},
        # The attention weights of one decoded token, added up for every position of 16 sequences.
        {"name": "weight_b16", "kind": "weight", "batch": 16, "tokens": 16, "past": 8000, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8"},
        # The same over a whole prompt.
        {"name": "weight_m2000", "kind": "weight", "batch": 1, "tokens": 2000, "past": 0, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "format": "int8"},
        # Eight sequences of up to 8100 positions cut to 4000: four first, 250 last, the heaviest between.
        {"name": "evict_b8", "kind": "evict", "batch": 8, "past": 8100, "kv_heads": 2, "head_dim": 128, "format": "int8",
         "budget": 4000, "sink": 4, "recent": 250},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["rope", "append", "attn", "attn", "attn", "weight", "evict"])
        d = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 2, 4, 8])
        case = {"kind": kind, "head_dim": d, "format": rng.choice(["int8", "int8", "e4m3"])}
        if kind == "rope":
            heads, table = rng.randint(1, 48), rng.choice(["given", "given", "none", "linear", "ntk", "parts"])
            case = {"kind": kind, "tokens": _log_int(rng, 1, 8000), "heads": heads, "row": heads + rng.choice([0, 0, 2, 7]),
                    "head_dim": d, "rotary": rng.choice([d, d, d // 2, d // 4]), "layout": rng.choice([HALF, INTERLEAVED]),
                    "dtype": rng.choice(["bf16", "bf16", "f32"]), "inverse": rng.random() < 0.25, "table": table,
                    "far": _log_int(rng, 8192, 1 << 17)}
        elif kind == "append":
            batch = _log_int(rng, 1, 64)
            rope = rng.random() < 0.7
            case |= {"batch": batch, "tokens": rng.choice([batch, _log_int(rng, batch, 6000)]), "past": _log_int(rng, 1, 2000) - 1,
                     "kv_heads": kv, "q_heads": kv * rng.randint(1, 8) if rope else 0, "rope": rope}
        elif kind in ("attn", "weight"):
            decode = rng.random() < 0.6
            batch = _log_int(rng, 1, 64) if decode else _log_int(rng, 1, 8)
            case |= {"batch": batch, "tokens": batch if decode else _log_int(rng, batch + 1, 4000),
                     "past": _log_int(rng, 1, 130000) - 1, "kv_heads": kv, "q_heads": kv * rng.randint(1, 16)}
        else:
            past = _log_int(rng, 100, 60000)
            budget = max(2, int(past * rng.uniform(0.2, 0.9)))
            sink = rng.randint(0, min(8, budget // 2))
            case |= {"batch": _log_int(rng, 1, 32), "past": past, "kv_heads": kv, "budget": budget, "sink": sink,
                     "recent": rng.randint(0, (budget - sink) // 2)}
        w = work(case)
        if w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES and _scores(case) <= LARGEST_SCORES:
            return case


# ---- sizes, from the case alone -----------------------------------------------------------

def _spread(i):
    return (0.37 + 0.6180339887 * i) % 1.0


def _counts(case):
    """New tokens of each sequence: one each, or a ragged split with an empty sequence and a single token in it."""
    b, t = case["batch"], case.get("tokens", 0)
    if t <= b:
        return [1] * b
    w = [0.1 + _spread(i) for i in range(b)]
    if b > 2:
        w[1] = w[2] = 0.0
    c = [int((t - 1) * x / sum(w)) for x in w]
    if b > 2:
        c[1] = 1
    c[0] += t - sum(c)
    return c


def _pasts(case):
    """Tokens of each sequence in the cache before: the first has the most, the others from half of that up."""
    return [case["past"] if i == 0 else int(case["past"] * (0.5 + 0.5 * _spread(i))) for i in range(case["batch"])]


def _lengths(case):
    return [p + c for p, c in zip(_pasts(case), _counts(case))] if case["kind"] != "evict" else _pasts(case)


def _ragged(case):
    return case["tokens"] > case["batch"]


def _max_ctx(case):
    return max(_lengths(case)) + 5  # not a whole number of blocks


def _rows(case):
    """(query, position) pairs of one head."""
    return sum(c * (n - c) + c * (c + 1) // 2 for c, n in zip(_counts(case), _lengths(case)))


def _scores(case):
    if case["kind"] not in ("attn", "weight"):
        return 0
    return case["batch"] * case["q_heads"] * max(_counts(case)) * max(_lengths(case))


def _span(case):
    """First slot, in blocks, that an append touches of each sequence, and the most blocks that it touches."""
    first = [p // BLOCK for p in _pasts(case)]
    return first, max(-(-n // BLOCK) - f for n, f in zip(_lengths(case), first))


def work(case):
    kind, d = case["kind"], case["head_dim"]
    if kind == "rope":
        x = case["tokens"] * case["heads"] * d * (2 if case["dtype"] == "bf16" else 4)
        table = case["tokens"] * case["rotary"] * 4
        return {"bytes": 2 * x + table * (2 if case["table"] != "given" else 1) + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    h = case["kv_heads"]
    if kind == "append":
        t, q = case["tokens"], case["q_heads"]
        _, blocks = _span(case)
        read = case["batch"] * blocks * BLOCK * h * d * 2 * 2  # bf16 keys and values of the touched blocks
        table = 4 * t * d if case["rope"] else 0
        return {"bytes": t * h * d * (4 + 4 + 2) + 4 * t * q * d + table + read, "flops": 6 * t * (h + q) * d}
    if kind == "evict":
        n, kept = sum(_lengths(case)), sum(min(x, case["budget"]) for x in _lengths(case))
        return {"bytes": 4 * n * h + kept * h * (2 * d + 2 * d + 4 + 4) + 4 * case["batch"] * case["budget"] * h * d, "flops": 4 * kept * h * d}
    n, t, q = sum(_lengths(case)), case["tokens"], case["q_heads"]
    if kind == "attn":
        return {"bytes": n * h * 2 * d + n * h // 4 + 4 * t * q * d + 4 * t * q, "flops": 4 * d * q * _rows(case)}
    return {"bytes": n * h * d + n * h // 8 + 8 * n * h + 2 * t * q * d + 4 * t * q, "flops": 2 * d * q * _rows(case)}


# ---- inputs -------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _codes(shape, form, g):
    """Bytes as quantised normal values leave them."""
    x = torch.randn(shape, device="cuda", generator=g)
    if form == "int8":
        return (x * 40.0).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    return (x * 140.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _cache(case, g):
    """A filled cache: keys and values of about N(0, 1), the scales of the blocks apart from each other."""
    b, h, d, ctx = case["batch"], case["kv_heads"], case["head_dim"], _max_ctx(case)
    blocks, gain = -(-ctx // BLOCK), 1 / 40.0 if case["format"] == "int8" else 1 / 140.0
    c = {"max_ctx": ctx, "format": case["format"]}
    for t in "kv":
        c[t] = _codes((b, h, blocks, BLOCK * d), case["format"], g)
        c[t + "_scale"] = gain * (0.75 + 0.5 * torch.rand((b, h, blocks), device="cuda", generator=g))
        c[t + "_open"] = _normal((b, h, BLOCK, d), g)
    return c


def _positions(case, g):
    return torch.randint(0, case["far"], (case["tokens"],), device="cuda", generator=g, dtype=torch.int32)


def _table64(positions, rotary, theta, scaling):
    """cos and sin of positions x frequencies in 64 bits: [positions, rotary / 2, 2]."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=positions.device)
    kind, factor, original = scaling["kind"], scaling["factor"], scaling["original"]
    if kind == "ntk" and rotary > 2:
        theta = theta * factor ** (rotary / (rotary - 2))
    f = torch.exp(-2.0 * i / rotary * math.log(theta))
    if kind == "linear":
        f = f / factor
    if kind == "parts":
        g = ((original * f / (2 * math.pi) - scaling["slow"]) / (scaling["fast"] - scaling["slow"])).clamp(0, 1)
        f = f * (g + (1 - g) / factor)
    a = positions.double()[:, None] * f
    return torch.stack([torch.cos(a), torch.sin(a)], -1) * scaling["gain"]


def _scaling(kind, far):
    """What stretches a context of 32768 to the positions in use."""
    factor = max(1.0, far / 32768.0) if kind not in ("given", "none") else 1.0
    return {"kind": "none" if kind == "given" else kind, "factor": factor, "original": 32768, "slow": 1.0, "fast": 32.0,
            "gain": 0.1 * math.log(factor) + 1.0 if kind == "parts" else 1.0}


def prepare(case, seed):
    g, kind, d = _gen(seed), case["kind"], case["head_dim"]
    s = {"case": case, "scale": 1.0 / math.sqrt(d)}
    if kind == "rope":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s["x"] = _normal((case["tokens"], case["row"], d), g, dt)[:, : case["heads"]]
        s["out"] = torch.empty((case["tokens"], case["heads"], d), dtype=dt, device="cuda")
        s["scaling"] = _scaling(case["table"], case["far"])
        if case["table"] == "given":
            s["positions"] = _positions(case, g)
            s["cos_sin"] = _table64(torch.arange(case["far"], device="cuda"), case["rotary"], THETA, s["scaling"]).float()
        else:  # consecutive positions, their own table: from the last of them backwards
            s["first"] = case["far"] - case["tokens"] if case["far"] > case["tokens"] else 0
            s["positions"] = torch.arange(case["tokens"], device="cuda", dtype=torch.int32)
        return s
    s["cache"] = _cache(case, g)
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    h = case["kv_heads"]
    if kind == "evict":
        b, n = case["batch"], s["cache"]["max_ctx"]
        w = torch.empty((b, h, n), device="cuda").exponential_(1.0, generator=g).pow_(4.0)  # a few heavy positions
        s["weight"] = torch.where(torch.rand((b, h, n), device="cuda", generator=g) < 0.1, 0.0, w)  # and many without any
        small = dict(case, past=case["budget"])
        s["to"] = _cache(small, g)
        s["to_weight"] = torch.zeros((b, h, s["to"]["max_ctx"]), device="cuda")
        s["kept"] = torch.zeros((b, h, case["budget"]), dtype=torch.int32, device="cuda")
        s["to_lengths"] = torch.zeros(b, dtype=torch.int32, device="cuda")
        return s
    t, counts = case["tokens"], _counts(case)
    if _ragged(case):
        ends = torch.tensor(counts, device="cuda").cumsum(0)
        s["starts"] = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    else:
        s["starts"] = None
    if kind == "append":
        s["k"], s["v"] = _normal((t, h, d), g), _normal((t, h, d), g)
        first, _ = _span(case)
        s["first"] = torch.tensor([BLOCK * f for f in first], dtype=torch.int32, device="cuda")
        s["open"] = s["cache"]["k_open"].clone(), s["cache"]["v_open"].clone()
        s["q"] = s["q_out"] = s["cos_sin"] = s["positions"] = None
        if case["rope"]:
            s["q"] = _normal((t, case["q_heads"], d), g)
            s["q_out"] = torch.empty_like(s["q"])
            n = _max_ctx(case)
            s["cos_sin"] = _table64(torch.arange(n, device="cuda"), d, THETA, _scaling("none", n)).float()
            s["positions"] = torch.cat([torch.arange(p, p + c) for p, c in zip(_pasts(case), counts)]).to("cuda", torch.int32)
        return s
    s["q"] = _normal((t, case["q_heads"], d), g) * 1.5
    if kind == "attn":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((t, case["q_heads"]), device="cuda")
        return s
    s["weight0"] = torch.rand((case["batch"], h, s["cache"]["max_ctx"]), device="cuda", generator=g)
    s["weight"] = s["weight0"].clone()
    s["lse"] = _plain_attention(s)[1]  # the attention call of the same step left it
    return s


# ---- the plain form -----------------------------------------------------------------------

def _values(codes, form):
    return codes.view(torch.int8).float() if form == "int8" else codes.view(torch.float8_e4m3fn).float()


def _read_keys(c, blocks=slice(None)):
    """f32 [batch, kv_heads, slots, head_dim] of a cache's keys."""
    k = c["k"][:, :, blocks]
    b, h, n, size = k.shape
    x = _values(k, c["format"]).view(b, h, n, size // BLOCK // 16, BLOCK, 16).transpose(3, 4).reshape(b, h, n, BLOCK, -1)
    return (x * c["k_scale"][:, :, blocks, None, None]).flatten(2, 3)


def _read_values(c, blocks=slice(None)):
    v = c["v"][:, :, blocks]
    b, h, n, size = v.shape
    x = _values(v, c["format"]).view(b, h, n, size // BLOCK // 32, 2, 32, 2, 2, 4)  # tile, h, dim, a, s, j
    x = x.permute(0, 1, 2, 7, 6, 4, 8, 3, 5).reshape(b, h, n, BLOCK, -1)
    return (x * c["v_scale"][:, :, blocks, None, None]).flatten(2, 3)


def _rotate(x, cs, layout, inverse=False):
    """x [tokens, heads, head_dim] turned by cs [tokens, rotary / 2, 2]."""
    r = 2 * cs.shape[1]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1] * (-1.0 if inverse else 1.0)
    x = x.float()
    if layout == HALF:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * c - b * n, a * n + b * c], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _of_tokens(s):
    """(sequence, place among its new tokens) of every token."""
    t = torch.arange(s["case"]["tokens"], device="cuda")
    if s["starts"] is None:
        return t, torch.zeros_like(t)
    b = torch.searchsorted(s["starts"][1:].contiguous(), t, right=True)
    return b, t - s["starts"].long()[b]


def _new_counts(s):
    return s["lengths"] * 0 + 1 if s["starts"] is None else s["starts"].diff()


def _quantise(x, form):
    """x [.., 32 slots, heads, head_dim] in one block: the values that its codes stand for, and its scale."""
    scale = x.abs().amax((-3, -1), keepdim=True) / (127.0 if form == "int8" else 448.0)
    q = torch.where(scale > 0, x / scale, 0.0)
    q = q.round().clamp(-127, 127) if form == "int8" else q.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return q * scale, scale[..., 0, :, 0]


def _plain_append(s):
    case, c, form = s["case"], s["cache"], s["case"]["format"]
    q, k = None, s["k"]
    if case["rope"]:
        cs = s["cos_sin"][s["positions"].long()]
        q, k = _rotate(s["q"], cs, HALF).to(torch.bfloat16), _rotate(k, cs, HALF).to(torch.bfloat16)
    seq, place = _of_tokens(s)
    lengths = s["lengths"].long()
    old = lengths - _new_counts(s).long()
    first, (_, blocks) = s["first"].long(), _span(case)
    batch = torch.arange(case["batch"], device="cuda")
    slots = first[:, None] + torch.arange(BLOCK * blocks, device="cuda")
    at = (old - first)[seq] + place
    last = (lengths - 1).clamp_min(0) // BLOCK  # the block whose raw rows are kept
    touched = (slots[:, ::BLOCK] < lengths[:, None]) & (lengths > old)[:, None]
    block = torch.where(touched, slots[:, ::BLOCK] // BLOCK, c["k"].shape[2])  # beyond the last: not written

    def one(new, raw, scales):
        x = torch.zeros((case["batch"], BLOCK * blocks, case["kv_heads"], case["head_dim"]), device="cuda")
        x[:, :BLOCK] = torch.where((slots[:, :BLOCK] < old[:, None])[..., None, None], raw.transpose(1, 2).float(), 0.0)
        x[seq, at] = new.float()
        y, scale = _quantise(x.unflatten(1, (blocks, BLOCK)), form)
        wide = torch.nn.functional.pad(scales, (0, 1))
        all_at = batch[:, None].expand_as(block)
        wide[all_at, :, block] = torch.where(touched[..., None], scale, wide[all_at, :, block])
        opened = raw.clone()
        mine = (old[seq] + place) // BLOCK == last[seq]
        row = torch.where(mine, (old[seq] + place) % BLOCK, BLOCK)
        padded = torch.nn.functional.pad(opened, (0, 0, 0, 1))
        padded[seq, :, row] = new
        return y.flatten(1, 2), wide[..., :-1], padded[:, :, :BLOCK]

    kv, ks, ko = one(k, s["open"][0], c["k_scale"])
    vv, vs, vo = one(s["v"], s["open"][1], c["v_scale"])
    # a sequence without new tokens keeps what it held: read from the cache
    there = (slots < lengths[:, None])
    idle = (lengths == old)[:, None, None, None]
    held = (slots // BLOCK).clamp_max(c["k"].shape[2] - 1)
    pick = held[:, ::BLOCK]
    few = {n: c[n][batch[:, None], :, pick].transpose(1, 2) for n in ("k", "v", "k_scale", "v_scale")} | {"format": form}
    kv = torch.where(idle, _read_keys(few).transpose(1, 2), kv)
    vv = torch.where(idle, _read_values(few).transpose(1, 2), vv)
    kv, vv = (torch.where(there[..., None, None], t, 0.0).to(torch.bfloat16) for t in (kv, vv))
    out = {"k": kv, "v": vv, "k_scale": ks, "v_scale": vs, "k_open": ko, "v_open": vo}
    return out | {"q": q} if q is not None else out


def _scores_of(s):
    """Scaled scores [batch, kv_heads, new tokens x group, slots] of the padded batch, -inf where a row does not look, and the places of the tokens in it."""
    case = s["case"]
    b, h, d, m = case["batch"], case["kv_heads"], case["head_dim"], max(_counts(case))
    group, n = case["q_heads"] // h, max(_lengths(case))
    seq, place = _of_tokens(s)
    q = torch.zeros((b, m, h, group, d), device="cuda")
    q[seq, place] = s["q"].float().view(-1, h, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(b, h, m * group, d)
    k = _read_keys(s["cache"], slice(0, -(-n // BLOCK)))[:, :, :n]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    counts = _new_counts(s)
    sees = (s["lengths"] - counts)[:, None] + torch.arange(m, device="cuda") + 1
    sees = torch.where(torch.arange(m, device="cuda") < counts[:, None], sees, 0)
    dark = torch.arange(n, device="cuda") >= sees[..., None]  # [batch, m, slots]
    x = x.view(b, h, m, group, n).masked_fill_(dark[:, None, :, None], -math.inf)
    return x, (seq, place)


def _plain_attention(s):
    case = s["case"]
    x, (seq, place) = _scores_of(s)
    b, h, m, group, n = x.shape
    top = x.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    v = _read_values(s["cache"], slice(0, -(-n // BLOCK)))[:, :, :n].contiguous()
    o = torch.matmul((p / total.clamp_min(1e-38)).view(b, h, m * group, n), v).view(b, h, m, group, -1)
    lse = (top + torch.log(total)).squeeze(-1)
    o, lse = o.permute(0, 2, 1, 3, 4)[seq, place], lse.permute(0, 2, 1, 3)[seq, place]
    return o.reshape(case["tokens"], case["q_heads"], -1).to(torch.bfloat16), lse.reshape(case["tokens"], case["q_heads"])


def _plain_weight(s):
    x, (seq, place) = _scores_of(s)
    b, h, m, group, n = x.shape
    lse = torch.full((b, m, h, group), math.inf, device="cuda")
    lse[seq, place] = s["lse"].view(-1, h, group)
    p = torch.exp(x - lse.permute(0, 2, 1, 3)[..., None]).sum((2, 3))
    slots, lengths = torch.arange(n, device="cuda"), s["lengths"][:, None, None]
    had = torch.where(slots < lengths - _new_counts(s)[:, None, None], s["weight0"][..., :n], 0.0)
    w = s["weight0"].clone()
    w[..., :n] = torch.where(slots < lengths, 0.98 * had + p, w[..., :n])
    return w


def _keep(s):
    """Kept slots in order [batch, kv_heads, budget] (a sequence that fits keeps all: its own slots, then none) and the new lengths."""
    case, w = s["case"], s["weight"]
    n, budget = s["lengths"].long()[:, None, None], case["budget"]
    at = torch.arange(w.shape[-1], device="cuda")
    rank = torch.where((at < case["sink"]) | (at >= n - case["recent"]), math.inf, w)
    rank = torch.where(at < n, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.sort(torch.where(order < n, order, w.shape[-1]), -1).values
    there = kept < n
    return torch.where(there, kept, 0), there, n.clamp_max(budget)


def _plain_evict(s):
    case, c, form, to = s["case"], s["cache"], s["case"]["format"], s["to"]
    kept, there, left = _keep(s)
    n = s["lengths"].long()[:, None, None]
    budget, last = case["budget"], (left - 1) // BLOCK
    blocks, d = -(-budget // BLOCK), case["head_dim"]
    pad = BLOCK * blocks - budget
    at = torch.arange(BLOCK * blocks, device="cuda")
    source, valid = torch.nn.functional.pad(kept, (0, pad)), torch.nn.functional.pad(there, (0, pad))
    fits = n <= budget
    raw = valid & (source // BLOCK == (n - 1) // BLOCK)  # rows of the last block are at hand as they came
    ends = (at // BLOCK == last) & ~fits  # rows of the new last block
    same = (~valid | (source == at)).unflatten(-1, (blocks, BLOCK)).all(-1, keepdim=True) & (fits | (torch.arange(blocks, device="cuda") != last))[..., None]

    def one(held, opened, scales, new_open, new_scales):
        x = torch.gather(held, 2, source[..., None].expand(-1, -1, -1, d))
        o = torch.gather(opened, 2, (source % BLOCK)[..., None].expand(-1, -1, -1, d)).float()
        y = torch.where(raw[..., None], o, x)
        y = torch.where(valid[..., None], torch.where(ends[..., None], y.to(torch.bfloat16).float(), y), 0.0)
        z, scale = _quantise(y.unflatten(2, (blocks, BLOCK)).unsqueeze(4), form)
        z, scale = z.squeeze(4), scale[..., 0]
        z = torch.where(same[..., None], x.unflatten(2, (blocks, BLOCK)), z).flatten(2, 3)
        scale = torch.where(same[..., 0], scales[..., :blocks], scale)
        row = torch.where(ends & valid, at % BLOCK, BLOCK)
        padded = torch.nn.functional.pad(new_open, (0, 0, 0, 1))
        padded.scatter_(2, row[..., None].expand(-1, -1, -1, d), y.to(torch.bfloat16))
        padded = torch.where(fits[..., None], torch.nn.functional.pad(opened, (0, 0, 0, 1)), padded)
        used = torch.arange(blocks, device="cuda") <= last
        all_scales = new_scales.clone()
        all_scales[..., :blocks] = torch.where(used, scale, all_scales[..., :blocks])
        z = torch.where(valid[..., None], z, 0.0)[:, :, :budget].transpose(1, 2)
        return z.to(torch.bfloat16), all_scales, padded[:, :, :BLOCK]

    k, ks, ko = one(_read_keys(c), c["k_open"], c["k_scale"], to["k_open"], to["k_scale"])
    v, vs, vo = one(_read_values(c), c["v_open"], c["v_scale"], to["v_open"], to["v_scale"])
    w = torch.zeros_like(s["to_weight"])
    w[..., :budget] = torch.where(there, torch.gather(s["weight"], 2, kept), 0.0)
    return {"kept": kept.to(torch.int32), "lengths": left.view(-1).to(torch.int32), "weight": w, "k": k, "v": v,
            "k_scale": ks, "v_scale": vs, "k_open": ko, "v_open": vo}


# ---- a pass -------------------------------------------------------------------------------

def _own_cache(kv8, c):
    return kv8.Kv8Cache.wrap(c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_open"], c["v_open"], c["max_ctx"],
                             kv8.INT8 if c["format"] == "int8" else kv8.E4M3)


def _run_own(s):
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kriya-rt_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kriya_q4 import kv8, rope

    case, kind = s["case"], s["case"]["kind"]
    if kind == "rope":
        cs = s.get("cos_sin")
        if cs is None:
            z = s["scaling"]
            cs = rope.table(case["rotary"], case["tokens"], THETA, first=s["first"],
                            scaling=rope.Scaling(z["kind"], z["factor"], z["original"], z["slow"], z["fast"], z["gain"]))
        y = rope.apply(s["x"], cs, s["positions"], layout=rope.HALF if case["layout"] == HALF else rope.INTERLEAVED,
                       inverse=case["inverse"], out=s["out"])
        return y if "cos_sin" in s else {"y": y, "table": cs}
    if "own" not in s:
        s["own"] = _own_cache(kv8, s["cache"])
        if kind == "attn":
            s["workspace"] = kv8.attention_workspace(s["own"], case["q_heads"], case["tokens"])
        if kind == "evict":
            s["own_to"] = _own_cache(kv8, s["to"])
    cache = s["own"]
    if kind == "append":
        if _ragged(case):  # the rows of the last block as they were before this pass
            cache.k_open.copy_(s["open"][0])
            cache.v_open.copy_(s["open"][1])
        kv8.append(cache, s["k"], s["v"], s["lengths"], starts=s["starts"], q=s["q"], q_out=s["q_out"],
                   cos_sin=s["cos_sin"], positions=s["positions"], layout=rope.HALF)
        k, v = kv8.dequant(cache, s["lengths"], BLOCK * _span(case)[1], first=s["first"])
        out = {"k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale, "k_open": cache.k_open, "v_open": cache.v_open}
        return out | {"q": s["q_out"]} if case["rope"] else out
    if kind == "attn":
        return kv8.attention(cache, s["q"], s["lengths"], starts=s["starts"], scale=s["scale"], out=s["out"], lse=s["lse"],
                             workspace=s["workspace"])
    if kind == "weight":
        s["weight"].copy_(s["weight0"])
        return kv8.accumulate_weight(cache, s["q"], s["lse"], s["lengths"], s["weight"], starts=s["starts"], scale=s["scale"],
                                     decay=0.98)
    kv8.evict(cache, s["lengths"], s["weight"], case["budget"], case["sink"], case["recent"], s["own_to"],
              s["to_weight"], s["kept"], s["to_lengths"])
    k, v = kv8.dequant(s["own_to"], s["to_lengths"], case["budget"])
    to = s["own_to"]
    return {"kept": s["kept"], "lengths": s["to_lengths"], "weight": s["to_weight"], "k": k, "v": v, "k_scale": to.k_scale,
            "v_scale": to.v_scale, "k_open": to.k_open, "v_open": to.v_open}


def run(s):
    if own:
        return _run_own(s)
    case, kind = s["case"], s["case"]["kind"]
    if kind == "rope":
        cs = s.get("cos_sin")
        if cs is None:
            cs = _table64(s["first"] + s["positions"], case["rotary"], THETA, s["scaling"]).float()
            y = _rotate(s["x"], cs, case["layout"], case["inverse"]).to(s["out"].dtype)
            return {"y": y, "table": cs}
        return _rotate(s["x"], cs[s["positions"].long()], case["layout"], case["inverse"]).to(s["out"].dtype)
    if kind == "append":
        return _plain_append(s)
    if kind == "attn":
        return _plain_attention(s)
    return _plain_weight(s) if kind == "weight" else _plain_evict(s)


# ---- the same in 64 bits, written apart: one sequence and head at a time ------------------

def _turn64(x, table, layout, inverse):
    x, r = x.double(), 2 * table.shape[1]
    z = torch.complex(table[..., 0].double(), table[..., 1].double())[:, None]
    z = z.conj() if inverse else z
    y = x.clone()
    if layout == HALF:
        w = torch.complex(x[..., : r // 2], x[..., r // 2: r]) * z
        y[..., : r // 2], y[..., r // 2: r] = w.real, w.imag
    else:
        w = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * z
        y[..., 0:r:2], y[..., 1:r:2] = w.real, w.imag
    return y


def _slots64(c, i, j, n, t):
    """Slots 0 .. n - 1 of sequence i, head j in 64 bits, from the layout's definition."""
    p = torch.arange(n, device="cuda")
    block, r = p // BLOCK, p % BLOCK
    codes = c[t][i, j]
    d = torch.arange(codes.shape[-1] // BLOCK, device="cuda")
    if t == "k":
        at = (d // 16) * (16 * BLOCK) + r[:, None] * 16 + d % 16
    else:
        at = (d // 32) * 1024 + (((r % 8) // 4) * 512)[:, None] + (d % 32) * 16 + ((r % 16) // 8 * 8 + r // 16 * 4 + r % 4)[:, None]
    return _values(codes[block[:, None], at], c["format"]).double() * c[t + "_scale"][i, j, block].double()[:, None]


def _coded64(x, form):
    """x [.., rows, head_dim] of one block and head: what its codes stand for, with the scale held in f32."""
    scale = (x.abs().amax((-2, -1), keepdim=True) / (127 if form == "int8" else 448)).float().double()
    q = torch.where(scale > 0, x / scale, 0.0)
    return (q.round() if form == "int8" else q.to(torch.float8_e4m3fn).double()) * scale, scale.flatten()


def exact(case, seed):
    s, kind, form = prepare(case, seed), case["kind"], case.get("format")

    def attention():
        h, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
        o = torch.empty((case["tokens"], case["q_heads"], case["head_dim"]), dtype=torch.float64, device="cuda")
        lse = torch.empty((case["tokens"], case["q_heads"]), dtype=torch.float64, device="cuda")
        mass = []
        t0 = 0
        for i, (c, n) in enumerate(zip(_counts(case), _lengths(case))):
            for j in range(h if c else 0):
                k, v = (_slots64(s["cache"], i, j, n, t) for t in "kv")
                q = s["q"][t0: t0 + c, j * group: (j + 1) * group].double().reshape(c * group, -1)
                x = q @ k.t() * s["scale"]
                limit = (n - c + 1 + torch.arange(c, device="cuda")).repeat_interleave(group)
                x.masked_fill_(torch.arange(n, device="cuda") >= limit[:, None], -math.inf)
                p = torch.softmax(x, -1)
                o[t0: t0 + c, j * group: (j + 1) * group] = (p @ v).view(c, group, -1)
                lse[t0: t0 + c, j * group: (j + 1) * group] = torch.logsumexp(x, -1).view(c, group)
                mass.append((i, j, n, c, p.sum(0)))
            t0 += c
        return o, lse, mass

    if kind == "rope":
        if case["table"] == "given":
            return _turn64(s["x"], s["cos_sin"][s["positions"].long()], case["layout"], case["inverse"])
        r, z, theta = case["rotary"], s["scaling"], THETA
        if z["kind"] == "ntk":
            theta *= z["factor"] ** (r / (r - 2))
        f = torch.tensor([theta ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
        if z["kind"] in ("linear", "parts"):
            turns = z["original"] * f / (2 * math.pi)
            g = ((turns - z["slow"]) / (z["fast"] - z["slow"])).clamp(0, 1) if z["kind"] == "parts" else 0.0
            f = g * f + (1 - g) * f / z["factor"]
        angle = (s["first"] + s["positions"].double())[:, None] * f
        table = z["gain"] * torch.view_as_real(torch.polar(torch.ones_like(angle), angle))
        return {"y": _turn64(s["x"], table, case["layout"], case["inverse"]), "table": table}
    if kind == "attn":
        return attention()[:2]
    if kind == "weight":
        w = s["weight0"].double()
        for i, j, n, c, p in attention()[2]:
            w[i, j, n - c: n] = 0.0
            w[i, j, :n] = 0.98 * w[i, j, :n] + p
        for i, (c, n) in enumerate(zip(_counts(case), _lengths(case))):
            if not c:
                w[i, :, :n] *= 0.98
        return w
    c, d = s["cache"], case["head_dim"]
    if kind == "append":
        k, q = s["k"].double(), None
        if case["rope"]:
            cs = s["cos_sin"][s["positions"].long()]
            q, k = (_turn64(x, cs, HALF, False) for x in (s["q"], s["k"]))
        out = {t: torch.zeros((case["batch"], BLOCK * _span(case)[1], case["kv_heads"], d), dtype=torch.float64, device="cuda") for t in "kv"}
        out |= {t + "_scale": c[t + "_scale"].double() for t in "kv"} | {t + "_open": c[t + "_open"].double() for t in "kv"}
        t0 = 0
        for i, (m, n, past) in enumerate(zip(_counts(case), _lengths(case), _pasts(case))):
            at = past // BLOCK * BLOCK
            for t, new in (("k", k), ("v", s["v"].double())):
                if not m:
                    for j in range(case["kv_heads"]):
                        out[t][i, : n - at, j] = _slots64(c, i, j, n, t)[at:]
                    continue
                x = torch.cat([c[t + "_open"][i, :, : past - at].double().transpose(0, 1), new[t0: t0 + m].to(torch.bfloat16).double()])
                for b in range(0, n - at, BLOCK):
                    y, scale = _coded64(x[b: b + BLOCK].transpose(0, 1), form)
                    out[t][i, b: b + y.shape[1]] = y.transpose(0, 1)
                    out[t + "_scale"][i, :, (at + b) // BLOCK] = scale.view(-1)
                rest = x[(n - 1) // BLOCK * BLOCK - at:]
                fresh = max(0, past - (n - 1) // BLOCK * BLOCK)
                out[t + "_open"][i, :, fresh: rest.shape[0]] = rest[fresh:].transpose(0, 1)
            t0 += m
        return out | {"q": q} if q is not None else out
    # evict: whole numbers by counting, values from the slots
    budget, to = case["budget"], s["to"]
    out = {"kept": None, "lengths": None, "weight": torch.zeros_like(s["to_weight"]).double()}
    out |= {t: torch.zeros((case["batch"], budget, case["kv_heads"], d), dtype=torch.float64, device="cuda") for t in "kv"}
    out |= {t + x: to[t + x].double() for x in ("_scale", "_open") for t in "kv"}
    for i, n in enumerate(_lengths(case)):
        for j in range(case["kv_heads"]):
            w, left = s["weight"][i, j, :n], min(n, budget)
            stay = torch.zeros(n, dtype=torch.bool, device="cuda")
            stay[: case["sink"]] = True
            stay[max(0, n - case["recent"]):] = True
            if n <= budget:
                stay[:] = True
            else:
                free = torch.nonzero(~stay).view(-1)
                best = free[torch.sort(w[free], descending=True, stable=True).indices[: budget - case["sink"] - case["recent"]]]
                stay[best] = True
            kept = torch.nonzero(stay).view(-1)
            out["weight"][i, j, :left] = w[kept].double()
            for t in "kv":
                held, raw = _slots64(c, i, j, n, t), c[t + "_open"][i, j].double()
                tail = (n - 1) // BLOCK * BLOCK
                for b in range(0, left, BLOCK):
                    rows = kept[b: b + BLOCK]
                    final = b + BLOCK >= left
                    if n <= budget or (not final and int(rows[-1]) == b + BLOCK - 1):
                        out[t][i, b: b + rows.numel(), j] = held[rows]
                        out[t + "_scale"][i, j, b // BLOCK] = c[t + "_scale"][i, j, b // BLOCK].double()
                        if final:
                            out[t + "_open"][i, j] = raw
                        continue
                    x = torch.where((rows >= tail)[:, None], raw[rows % BLOCK], held[rows])
                    if final:
                        x = x.float().to(torch.bfloat16).double()
                        out[t + "_open"][i, j, : rows.numel()] = x
                    y, scale = _coded64(x, form)
                    out[t][i, b: b + rows.numel(), j] = y
                    out[t + "_scale"][i, j, b // BLOCK] = scale.view(())
    return out
