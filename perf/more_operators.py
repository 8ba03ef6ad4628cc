"""A paged key/value cache and the trees of drafted tokens that are verified over it: the calls of a server that shares one
pool of pages among its sequences, each in a plain form (elementary torch operations) and as kriya_q4 offers it.

A pool holds pages of `page` slots (16, 32, 64 ..) in bf16, [layers, pages, kv_heads, page / 16, 16 * head_dim], and a table
names the page of every `page` slots of a sequence (-1: none). The 16 slots of a unit stand in the order of the matrix
instructions' operands: keys as [head_dim / 8][16 slots][8], values as [head_dim / 32][2 h][32 dims][2 a][4 j] with
slot 8 a + 4 h + j.
"""
import math
import os
import random
import sys

import torch

own = False

UNIT = 16
THETA = 1e6
EPS = 1e-6
VOCAB = 151936
LARGEST_FLOPS = 6e10  # of a drawn case; the largest listed one has more
LARGEST_BYTES = 4e8
LARGEST_SCORES = 2.4e8  # scores of the plain attention held at once, in elements


def listed():
    return [
        # The new token of 16 sequences: rotated into its page, q beside it.
        {"name": "append_b16", "kind": "append", "batch": 16, "tokens": 16, "past": 511, "page": 16, "kv_heads": 2,
         "q_heads": 16, "head_dim": 128, "rope": True, "norm": False},
        # The prompts of five sequences in one ragged batch, one of them half in the cache, one empty; heads normalised.
        {"name": "append_m3907", "kind": "append", "batch": 5, "tokens": 3907, "past": 1000, "page": 32, "kv_heads": 8,
         "q_heads": 32, "head_dim": 64, "rope": True, "norm": True},
        # One decoded token of five sequences of different lengths up to 3000: the smallest attention call.
        {"name": "attn_b5", "kind": "attn", "batch": 5, "tokens": 5, "past": 2999, "page": 16, "kv_heads": 2, "q_heads": 16,
         "head_dim": 128, "tree": False},
        # A large decode batch: 48 sequences up to 8000 positions, few heads to share each row.
        {"name": "attn_b48", "kind": "attn", "batch": 48, "tokens": 48, "past": 7999, "page": 64, "kv_heads": 8,
         "q_heads": 32, "head_dim": 64, "tree": False},
        # One sequence with a very long context.
        {"name": "attn_b1_long", "kind": "attn", "batch": 1, "tokens": 1, "past": 131071, "page": 128, "kv_heads": 2,
         "q_heads": 16, "head_dim": 128, "tree": False},
        # A whole prompt, causal: 3907 tokens, a ragged last tile.
        {"name": "attn_m3907", "kind": "attn", "batch": 1, "tokens": 3907, "past": 0, "page": 16, "kv_heads": 2,
         "q_heads": 16, "head_dim": 128, "tree": False},
        # A step that mixes chunks of prompts with decoded tokens (one sequence has a single new token, one has none).
        {"name": "attn_chunk", "kind": "attn", "batch": 4, "tokens": 600, "past": 12000, "page": 32, "kv_heads": 2,
         "q_heads": 10, "head_dim": 256, "tree": False},
        # Trees of about 30 drafted tokens verified in 8 sequences.
        {"name": "tree_b8", "kind": "attn", "batch": 8, "tokens": 250, "past": 5000, "page": 16, "kv_heads": 2,
         "q_heads": 16, "head_dim": 128, "tree": True},
        # One sequence's tree planned: the smallest call.
        {"name": "plan_b1", "kind": "plan", "batch": 1, "tokens": 24, "past": 900},
        # The trees of a large batch, of up to some hundred nodes.
        {"name": "plan_b64", "kind": "plan", "batch": 64, "tokens": 4100, "past": 3000},
        # What a small model's step keeps of the trees of four sequences: all layers at once.
        {"name": "commit_b4", "kind": "commit", "batch": 4, "tokens": 50, "past": 60, "page": 16, "kv_heads": 2,
         "head_dim": 128, "layers": 36, "max_path": 8},
        # The same for a large batch and larger trees.
        {"name": "commit_b48", "kind": "commit", "batch": 48, "tokens": 2900, "past": 120, "page": 32, "kv_heads": 8,
         "head_dim": 64, "layers": 24, "max_path": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "append", "attn", "attn", "attn", "tree", "tree", "plan", "commit"])
        case = {"kind": kind, "page": rng.choice([16, 16, 32, 64, 128, 256]), "head_dim": rng.choice([64, 64, 96, 128, 128, 128, 192, 256]),
                "kv_heads": rng.choice([1, 2, 2, 4, 8])}
        kv, batch = case["kv_heads"], _log_int(rng, 1, 64)
        if kind == "append":
            case |= {"batch": batch, "tokens": rng.choice([batch, _log_int(rng, batch, 6000)]), "past": _log_int(rng, 1, 4000) - 1,
                     "q_heads": kv * rng.randint(1, 8), "rope": rng.random() < 0.8, "norm": rng.random() < 0.5}
        elif kind == "attn":
            decode = rng.random() < 0.6
            batch = batch if decode else _log_int(rng, 1, 8)
            case |= {"batch": batch, "tokens": batch if decode else _log_int(rng, batch + 1, 4000), "tree": False,
                     "past": _log_int(rng, 1, 130000) - 1, "q_heads": kv * rng.randint(1, 16)}
        elif kind == "tree":
            case |= {"kind": "attn", "batch": batch, "tokens": batch * rng.randint(2, 70), "tree": True, "past": _log_int(rng, 1, 30000) - 1,
                     "q_heads": kv * rng.randint(1, 16)}
        elif kind == "plan":
            case = {"kind": kind, "batch": batch, "tokens": batch * rng.randint(2, 130), "past": _log_int(rng, 1, 100000) - 1}
        else:
            case |= {"batch": batch, "tokens": batch * rng.randint(2, 70), "past": _log_int(rng, 1, 200) - 1,
                     "layers": rng.randint(1, 36), "max_path": rng.randint(1, 20)}
        w = work(case)
        if (w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES and _scores(case) <= LARGEST_SCORES
                and (case["kind"] != "commit" or _pool_bytes(case) <= 1.2e9)):
            return case


# ---- sizes, from the case alone -----------------------------------------------------------

def _spread(i):
    return (0.37 + 0.6180339887 * i) % 1.0


def _drafted(case):
    return case["kind"] in ("plan", "commit") or case.get("tree", False)


def _counts(case):
    """New tokens of each sequence: one each; of prompts a ragged split with an empty sequence and a single token in it; of
    trees a split with every size from half of the mean up."""
    b, t = case["batch"], case["tokens"]
    if t <= b:
        return [1] * b
    w = [(1.0 if _drafted(case) else 0.1) + _spread(i) for i in range(b)]
    if b > 2 and not _drafted(case):
        w[1] = w[2] = 0.0
    c = [int((t - 1) * x / sum(w)) for x in w]
    if _drafted(case):
        c = [max(1, x) for x in c]
    elif b > 2:
        c[1] = 1
    c[0] += t - sum(c)
    if c[0] < 1:
        return [t // b + (1 if i < t % b else 0) for i in range(b)]
    return c


def _pasts(case):
    """Tokens of each sequence in the cache before: the first has the most, the others from half of that up."""
    return [case["past"] if i == 0 else int(case["past"] * (0.5 + 0.5 * _spread(i))) for i in range(case["batch"])]


def _lengths(case):
    return [p + c for p, c in zip(_pasts(case), _counts(case))]


def _words(case):
    return -(-max(_counts(case)) // 32)


def _pairs(case):
    """(query, position) pairs of one head; of a tree at least its own node each."""
    inner = (lambda c: c) if _drafted(case) else (lambda c: c * (c + 1) // 2)
    return sum(c * (n - c) + inner(c) for c, n in zip(_counts(case), _lengths(case)))


def _scores(case):
    if case["kind"] != "attn":
        return 0
    return case["batch"] * case["q_heads"] * max(_counts(case)) * max(_lengths(case))


def _pages(case):
    """Pages of each sequence's table, and of the pool: a few are nobody's."""
    each = [-(-n // case["page"]) for n in _lengths(case)]
    return each, sum(each) + 3


def _pool_bytes(case):
    return 4 * case.get("layers", 1) * _pages(case)[1] * case["page"] * case["kv_heads"] * case["head_dim"]


def work(case):
    t = case["tokens"]
    if case["kind"] == "plan":
        return {"bytes": 4 * t * (2 + _words(case)) + 8 * case["batch"], "flops": 0}
    d, h = case["head_dim"], case["kv_heads"]
    if case["kind"] == "commit":
        moved = case["batch"] * min(case["max_path"] - 1, 3)  # about what is accepted beyond the first nodes
        return {"bytes": 12 * t + 4 * case["batch"] * (case["max_path"] + 4) + 8 * moved * case["layers"] * h * d, "flops": 0}
    q = case["q_heads"]
    if case["kind"] == "append":
        return {"bytes": t * d * (8 * h + 4 * q + (4 if case["rope"] else 0)) + 8 * t,
                "flops": t * (h + q) * d * ((3 if case["rope"] else 0) + (4 if case["norm"] else 0))}
    n = sum(_lengths(case))
    return {"bytes": 4 * n * h * d + 4 * t * q * (d + 1) + (4 * t * _words(case) if case["tree"] else 0), "flops": 4 * d * q * _pairs(case)}


# ---- inputs -------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case, rng):
    """The pages of the sequences, scattered over the pool as they were taken and given back; -1 behind the last."""
    each, total = _pages(case)
    order = list(range(total))
    rng.shuffle(order)
    rows, at = [], 0
    for n in each:
        rows.append(order[at: at + n] + [-1] * (max(each) - n + 1))
        at += n
    return _int32(rows)


def _trees(case, rng):
    """Parents of each sequence's nodes (-1 for node 0, the token that was sampled last): runs and branches."""
    def tree(m):
        return [-1] + [i - 1 if rng.random() < 0.45 else rng.randrange(max(0, i - 8), i) for i in range(1, m)]
    return [tree(m) for m in _counts(case)]


def _choices(parents, rng, most):
    """Drafted tokens of a tree, and the model's choices after each: on one way down from node 0 they are the children's tokens."""
    tokens = [rng.randrange(VOCAB - 1) for _ in parents]
    targets = [rng.randrange(VOCAB - 1) for _ in parents]
    for i in range(2, len(parents)):  # now and then two children with the same token: the first one counts
        if parents[i] == parents[i - 1] and rng.random() < 0.1:
            tokens[i] = tokens[i - 1]
    at, left = 0, rng.randint(0, most)
    while left:
        children = [i for i, p in enumerate(parents) if p == at]
        if not children:
            break
        child = rng.choice(children)
        targets[at] = tokens[child]
        at, left = next(i for i in children if tokens[i] == tokens[child]), left - 1
    targets[at] = VOCAB - 1
    return tokens, targets


def prepare(case, seed):
    g, rng, kind = _gen(seed), random.Random(seed), case["kind"]
    counts, t = _counts(case), case["tokens"]
    s = {"case": case, "lengths": _int32(_lengths(case)), "starts": None}
    if t > case["batch"] or _drafted(case):
        s["starts"] = _int32([sum(counts[:i]) for i in range(case["batch"] + 1)])
    if _drafted(case):
        trees = _trees(case, rng)
        s["parents"] = _int32([p for x in trees for p in x])
    if kind == "plan":
        s["mask"] = torch.empty((t, _words(case)), dtype=torch.int32, device="cuda")
        s["positions"] = torch.empty(t, dtype=torch.int32, device="cuda")
        return s
    d, h = case["head_dim"], case["kv_heads"]
    s["table"], s["scale"] = _table(case, rng), 1.0 / math.sqrt(d)
    shape = (case.get("layers", 1), _pages(case)[1], h, case["page"] // UNIT, UNIT * d)
    s["k"], s["v"] = _normal(shape, g), _normal(shape, g)
    if kind == "commit":
        choices = [_choices(x, rng, 7) for x in trees]
        s["tokens"], s["targets"] = (_int32([v for c in choices for v in c[i]]) for i in (0, 1))
        s["path"] = torch.zeros((case["batch"], case["max_path"]), dtype=torch.int32, device="cuda")
        s["counts"], s["next"], s["new_lengths"] = (torch.zeros_like(s["lengths"]) for _ in range(3))
        return s
    q = case["q_heads"]
    s["q"] = _normal((t, q, d), g)
    if kind == "append":
        s["new_k"], s["new_v"], s["q_out"] = _normal((t, h, d), g), _normal((t, h, d), g), torch.empty_like(s["q"])
        s["q_norm"] = s["k_norm"] = s["cos_sin"] = s["positions"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1.0 + 0.1 * _normal(2 * d, g, torch.float32)).to(torch.bfloat16).view(2, d)
        if case["rope"]:
            rows = max(_lengths(case))
            f = torch.exp(torch.arange(d // 2, device="cuda").double() * (-2.0 / d * math.log(THETA)))
            a = torch.arange(rows, device="cuda").double()[:, None] * f
            s["cos_sin"] = torch.stack([a.cos(), a.sin()], -1).float()
            s["positions"] = torch.cat([torch.arange(p, p + c) for p, c in zip(_pasts(case), counts)]).to("cuda", torch.int32)
        return s
    s["q"] = s["q"] * 1.5
    s["out"], s["lse"], s["mask"] = torch.empty_like(s["q"]), torch.empty((t, q), device="cuda"), None
    if case["tree"]:
        s["mask"] = _plain_plan(s)["mask"]  # the step planned it before its first layer
    return s


# ---- the plain form -----------------------------------------------------------------------

def _of_tokens(s):
    """(sequence, place among its new tokens) of every token, and new tokens of every sequence."""
    t = torch.arange(s["case"]["tokens"], device="cuda")
    if s["starts"] is None:
        return t, torch.zeros_like(t), torch.ones_like(t)
    starts = s["starts"].long()
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return b, t - starts[b], starts.diff()


def _ancestors(s, seq, place):
    """[batch, nodes, nodes]: 1 where a node is the other's ancestor or itself. With A the matrix of parents, strictly lower
    triangular, that is 1 + A + A^2 + .. = (1 - A)^-1."""
    b, m = s["case"]["batch"], max(_counts(s["case"]))
    a = torch.eye(m, device="cuda").repeat(b, 1, 1)
    p = s["parents"].long()
    a[seq, place, p.clamp_min(0)] -= torch.where(p >= 0, 1.0, 0.0)
    return torch.linalg.solve_triangular(a, torch.eye(m, device="cuda").expand_as(a), upper=False, unitriangular=True)


def _plain_plan(s):
    seq, place, counts = _of_tokens(s)
    up = _ancestors(s, seq, place)[seq, place]
    words = _words(s["case"])
    bits = torch.nn.functional.pad(up, (0, 32 * words - up.shape[1])).long().view(-1, words, 32)
    mask = (bits << torch.arange(32, device="cuda")).sum(-1)
    first = s["lengths"].long() - counts
    return {"mask": torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32),
            "positions": (first[seq] + up.sum(-1).long() - 1).to(torch.int32)}


def _key_view(pool, d):
    return pool.view(*pool.shape[:-1], d // 8, UNIT, 8)


def _value_view(pool, d):
    return pool.view(*pool.shape[:-1], d // 32, 2, 32, 2, 4)


def _place(s, seq, slots):
    """(page, unit of it, slot of that) of slots of sequences."""
    size = s["case"]["page"]
    return s["table"].long()[seq, slots // size], slots % size // UNIT, slots % UNIT


def _read(s, n):
    """f32 keys and values [batch, kv_heads, n, head_dim] of the first slots."""
    d, pages = s["case"]["head_dim"], s["table"][:, : -(-n // s["case"]["page"])].long().clamp_min(0)
    k, v = _key_view(s["k"][0][pages], d), _value_view(s["v"][0][pages], d)  # [batch, page, head, unit, ..]
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(k.shape[0], k.shape[2], -1, d)
    v = v.permute(0, 2, 1, 3, 7, 5, 8, 4, 6).reshape(v.shape[0], v.shape[2], -1, d)
    return k[:, :, :n].float(), v[:, :, :n].float()


def _turned(x, weight, s):
    """Heads x [tokens, heads, head_dim] normalised and rotated, in f32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    if s["cos_sin"] is not None:
        cs = s["cos_sin"][s["positions"].long()][:, None]
        a, b = x.chunk(2, -1)
        x = torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)
    return x.to(torch.bfloat16)


def _plain_append(s):
    d = s["case"]["head_dim"]
    seq, place, counts = _of_tokens(s)
    page, unit, r = _place(s, seq, (s["lengths"].long() - counts)[seq] + place)
    k = _turned(s["new_k"], s["k_norm"], s)
    _key_view(s["k"][0], d)[page, :, unit, :, r] = k.unflatten(-1, (d // 8, 8))
    _value_view(s["v"][0], d)[page, :, unit, :, r % 8 // 4, :, r // 8, r % 4] = s["new_v"].unflatten(-1, (d // 32, 32))
    out = {"k": s["k"], "v": s["v"]}
    return out | {"q": _turned(s["q"], s["q_norm"], s)} if s["case"]["rope"] or s["case"]["norm"] else out


def _plain_attention(s):
    case = s["case"]
    b, h, d, m, n = case["batch"], case["kv_heads"], case["head_dim"], max(_counts(case)), max(_lengths(case))
    group = case["q_heads"] // h
    seq, place, counts = _of_tokens(s)
    q = torch.zeros((b, m, h, group, d), device="cuda")
    q[seq, place] = s["q"].float().view(-1, h, group, d)
    k, v = _read(s, n)
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(b, h, m * group, d), k.transpose(2, 3).contiguous()) * s["scale"]
    slots, first = torch.arange(n, device="cuda"), (s["lengths"].long() - counts)[:, None, None]
    node = slots - first  # [batch, 1, slots]: place among the new tokens
    if s["mask"] is None:
        sees = node <= torch.arange(m, device="cuda")[:, None]
    else:
        words = torch.zeros((b, m, s["mask"].shape[1]), dtype=torch.int64, device="cuda")
        words[seq, place] = s["mask"].long()
        at = node.clamp(0, 32 * words.shape[2] - 1).expand(b, m, n)
        sees = (node < 0) | ((torch.gather(words, 2, at // 32) >> (at % 32) & 1 > 0) & (node < counts[:, None, None]))
    x = x.view(b, h, m, group, n).masked_fill_(~sees[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / total.clamp_min(1e-38)).view(b, h, m * group, n), v.contiguous()).view(b, h, m, group, d)
    lse = (top + torch.log(total)).squeeze(-1)
    o, lse = o.permute(0, 2, 1, 3, 4)[seq, place], lse.permute(0, 2, 1, 3)[seq, place]
    return o.reshape(case["tokens"], case["q_heads"], d).to(torch.bfloat16), lse.reshape(case["tokens"], case["q_heads"])


def _plain_commit(s):
    case = s["case"]
    b, m, d, most = case["batch"], max(_counts(case)), case["head_dim"], case["max_path"]
    seq, place, counts = _of_tokens(s)
    up = _ancestors(s, seq, place)
    parent = torch.full((b, m), -1, device="cuda")
    token, target = torch.full((b, m), -1, device="cuda"), torch.full((b, m), -2, device="cuda")
    parent[seq, place], token[seq, place], target[seq, place] = s["parents"].long(), s["tokens"].long(), s["targets"].long()
    # a node follows its parent where it has the token chosen there, and no sibling before it has
    fits = (parent >= 0) & (token == torch.gather(target, 1, parent.clamp_min(0)))
    twin = (parent[:, :, None] == parent[:, None, :]) & fits[:, :, None] & fits[:, None, :]
    fits &= ~torch.tril(twin, -1).any(-1)
    fits[:, 0] = True
    off = torch.matmul(up, (~fits).float()[..., None].contiguous())[..., 0]
    taken = (off == 0) & (torch.arange(m, device="cuda") < counts[:, None]) & (up.sum(-1) <= most)
    path = torch.sort(torch.where(taken, torch.arange(m, device="cuda"), m), 1).values
    path = torch.nn.functional.pad(path, (0, max(0, most - m)), value=m)[:, :most]
    there = path < m
    kept = there.sum(1)
    path = torch.where(there, path, 0)
    last = torch.gather(path, 1, (kept - 1)[:, None])
    first = s["lengths"].long() - counts
    of = torch.arange(b, device="cuda")[:, None].expand(-1, most)
    source = _place(s, of, first[:, None] + path)
    to = _place(s, of, first[:, None] + torch.where(there, torch.arange(most, device="cuda"), 0))
    k, v = _key_view(s["k"], d), _value_view(s["v"], d)
    page, unit, r = source
    rows = k[:, page, :, unit, :, r], v[:, page, :, unit, :, r % 8 // 4, :, r // 8, r % 4]
    page, unit, r = to
    k[:, page, :, unit, :, r], v[:, page, :, unit, :, r % 8 // 4, :, r // 8, r % 4] = rows
    return {"k": s["k"], "v": s["v"], "path": path.to(torch.int32), "counts": kept.to(torch.int32),
            "next": torch.gather(target, 1, last)[:, 0].to(torch.int32), "lengths": (first + kept).to(torch.int32)}


# ---- a pass -------------------------------------------------------------------------------

def _run_own(s):
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kriya-rt_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from kriya_q4 import paged

    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        mask, positions = paged.tree_plan(s["parents"], s["lengths"], s["starts"], mask=s["mask"], positions=s["positions"])
        return {"mask": mask, "positions": positions}
    if "own" not in s:
        s["own"] = paged.PagedCache.wrap(s["k"], s["v"])
        s["step"] = paged.Step(s["table"], s["lengths"], s["starts"])
        if kind == "attn":
            s["workspace"] = paged.attention_workspace(s["own"], s["step"], case["q_heads"], case["tokens"])
    cache, step = s["own"], s["step"]
    if kind == "append":
        turned = case["rope"] or case["norm"]
        paged.append(cache, step, s["new_k"], s["new_v"], q=s["q"] if turned else None, q_out=s["q_out"] if turned else None,
                     cos_sin=s["cos_sin"], positions=s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return {"k": s["k"], "v": s["v"], "q": s["q_out"]} if turned else {"k": s["k"], "v": s["v"]}
    if kind == "attn":
        return paged.attention(cache, step, s["q"], mask=s["mask"], scale=s["scale"], out=s["out"], lse=s["lse"], workspace=s["workspace"])
    paged.commit(cache, step, s["tokens"], s["parents"], s["targets"], s["path"], s["counts"], s["next"], s["new_lengths"])
    return {"k": s["k"], "v": s["v"], "path": s["path"], "counts": s["counts"], "next": s["next"], "lengths": s["new_lengths"]}


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "plan":
        return _plain_plan(s)
    if kind == "append":
        return _plain_append(s)
    return _plain_attention(s) if kind == "attn" else _plain_commit(s)


# ---- the same in 64 bits, written apart: one sequence and head at a time ------------------

def _at64(d, r, which):
    """Places in a unit of all dims of its slots r [..]: [.., d], from the layout's definition."""
    x = torch.arange(d, device="cuda")
    if which == "k":
        return x // 8 * (8 * UNIT) + r[..., None] * 8 + x % 8
    return x // 32 * 512 + (r % 8 // 4 * 256 + r // 8 * 4 + r % 4)[..., None] + x % 32 * 8


def _flat64(s, i, head, slots, which, layer=0):
    """Flat places in the pool of all dims of a sequence's slots."""
    pool, size, d = s[which], s["case"]["page"], s["case"]["head_dim"]
    pages = s["table"][i].long()[slots // size]
    unit = ((layer * pool.shape[1] + pages) * pool.shape[2] + head) * pool.shape[3] + slots % size // UNIT
    return unit[:, None] * (UNIT * d) + _at64(d, slots % UNIT, which)


def _turned64(x, weight, s):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    if s["cos_sin"] is not None:
        z = torch.view_as_complex(s["cos_sin"][s["positions"].long()].double().contiguous())[:, None]
        half = x.shape[-1] // 2
        y = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * z
        x = torch.cat([y.real, y.imag], -1)
    return x


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers only
    s, kind, d, h = prepare(case, seed), case["kind"], case["head_dim"], case["kv_heads"]
    spans = list(zip(_counts(case), _lengths(case)))
    if kind == "append":
        k, v = s["k"].double(), s["v"].double()
        new = {"k": _turned64(s["new_k"], s["k_norm"], s), "v": s["new_v"].double()}
        t0 = 0
        for i, (c, n) in enumerate(spans):
            slots = torch.arange(n - c, n, device="cuda")
            for j in range(h):
                for name, pool in (("k", k), ("v", v)):
                    pool.view(-1)[_flat64(s, i, j, slots, name).flatten()] = new[name][t0: t0 + c, j].flatten()
            t0 += c
        out = {"k": k, "v": v}
        return out | {"q": _turned64(s["q"], s["q_norm"], s)} if case["rope"] or case["norm"] else out
    parents = s["parents"].tolist() if _drafted(case) else None
    if kind == "attn":
        group = case["q_heads"] // h
        o = torch.empty((case["tokens"], case["q_heads"], d), dtype=torch.float64, device="cuda")
        lse = torch.empty((case["tokens"], case["q_heads"]), dtype=torch.float64, device="cuda")
        t0 = 0
        for i, (c, n) in enumerate(spans):
            sees = torch.ones((c, n), dtype=torch.bool)
            if parents is None:
                sees = sees.tril(n - c)
            else:
                sees[:, n - c:] = False
                for a in range(c):
                    if parents[t0 + a] >= 0:
                        sees[a, n - c:] = sees[parents[t0 + a], n - c:]
                    sees[a, n - c + a] = True
            sees = sees.to("cuda")
            for j in range(h if c else 0):
                k, v = (s[w].view(-1)[_flat64(s, i, j, torch.arange(n, device="cuda"), w)].double() for w in "kv")
                q = s["q"][t0: t0 + c, j * group: (j + 1) * group].double()
                x = torch.matmul(q.reshape(c * group, d), k.t()).view(c, group, n) * s["scale"]
                x = torch.where(sees[:, None], x, -math.inf)
                o[t0: t0 + c, j * group: (j + 1) * group] = torch.matmul(torch.softmax(x, -1).view(c * group, n), v).view(c, group, d)
                lse[t0: t0 + c, j * group: (j + 1) * group] = torch.logsumexp(x, -1)
            t0 += c
        return o, lse
    k, v = s["k"].double(), s["v"].double()
    tokens, targets = s["tokens"].tolist(), s["targets"].tolist()
    t0 = 0
    for i, (c, n) in enumerate(spans):
        path = [0]
        while len(path) < case["max_path"]:
            following = [j for j in range(c) if parents[t0 + j] == path[-1] and tokens[t0 + j] == targets[t0 + path[-1]]]
            if not following:
                break
            path.append(following[0])
        old, new = n - c + torch.tensor(path, device="cuda"), n - c + torch.arange(len(path), device="cuda")
        for name, pool in (("k", k), ("v", v)):
            layer = pool[0].numel()
            heads = torch.arange(h, device="cuda")[:, None, None] * (pool.shape[3] * UNIT * d)
            flat = pool.view(pool.shape[0], layer)
            rows = flat[:, (_flat64(s, i, 0, old, name) + heads).flatten()]
            flat[:, (_flat64(s, i, 0, new, name) + heads).flatten()] = rows
        t0 += c
    return {"k": k, "v": v, "path": None, "counts": None, "next": None, "lengths": None}
