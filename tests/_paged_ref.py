"""The paged cache, its attention, and the plan and commit of trees in 64 bits on the CPU, from include/kriya_paged.h alone."""
import math

import torch

UNIT = 16


def key_at(r, d):
    return d // 8 * 128 + r * 8 + d % 8


def value_at(r, d):
    return d // 32 * 512 + r // 4 % 2 * 256 + d % 32 * 8 + r // 8 * 4 + r % 4


def _order(d, at):
    return at(torch.arange(UNIT)[:, None], torch.arange(d)[None])


def slots_of(pool, which, pages, page):
    """Slots of one layer's pages (a list; None: zeros) in order, f64 [kv_heads, slots, head_dim]."""
    d = pool.shape[-1] // UNIT
    order = _order(d, key_at if which == "k" else value_at)
    out = []
    for p in pages:
        x = torch.zeros(pool.shape[1:], dtype=pool.dtype) if p is None else pool[p].cpu()
        out.append(x[..., order].flatten(1, 2).double())
    return torch.cat(out, 1)


def spans(starts, lengths):
    """[(first row, new tokens, length)] of every sequence."""
    n = [int(x) for x in lengths]
    if starts is None:
        return [(b, 1, x) for b, x in enumerate(n)]
    s = [int(x) for x in starts]
    return [(s[b], s[b + 1] - s[b], x) for b, x in enumerate(n)]


def sees(m, n, slots, mask=None):
    """bool [m, slots]: what the new tokens of a sequence see; mask: rows of whole numbers (words of 32 bits) or None."""
    out = torch.zeros(m, slots, dtype=torch.bool)
    for i in range(m):
        for p in range(min(n, slots)):
            j = p - (n - m)
            if mask is None:
                out[i, p] = j <= i
            else:
                out[i, p] = j < 0 or (j // 32 < len(mask[i]) and (int(mask[i][j // 32]) >> (j % 32)) & 1 == 1)
    return out


def attention(q, k, v, seen, scale):
    """One sequence: q [m, heads, d], k, v f64 [kv, slots, d], seen [m, slots] -> out, lse, and for bounds sum p |v|, max sum |q k|."""
    m, heads, d = q.shape
    group = heads // k.shape[0]
    out = torch.zeros(m, heads, d, dtype=torch.float64)
    lse = torch.full((m, heads), -math.inf, dtype=torch.float64)
    mass, terms = torch.zeros_like(out), torch.zeros_like(lse)
    q = q.double()
    for i in range(m):
        at = seen[i].nonzero().view(-1)
        if not at.numel():
            continue
        for h in range(heads):
            kk, vv = k[h // group][at], v[h // group][at]
            x = kk @ q[i, h] * scale
            p = torch.softmax(x, 0)
            out[i, h], mass[i, h] = p @ vv, p @ vv.abs()
            lse[i, h] = torch.logsumexp(x, 0)
            terms[i, h] = (kk.abs() @ q[i, h].abs()).max() * abs(scale)
    return out, lse, mass, terms


def plan(parents, n, words):
    """(mask rows, positions) of one sequence's nodes."""
    m, rows, positions = len(parents), [], []
    for i in range(m):
        bits, depth, at = 0, 0, i
        if i >= 32 * words:
            rows.append([0] * words)
            positions.append(n - m)
            continue
        while at is not None:
            bits |= 1 << at
            depth += 1
            at = parents[at] if 0 <= parents[at] < at else None
        rows.append([bits >> (32 * w) & 0xFFFFFFFF for w in range(words)])
        positions.append(n - m + depth - 1)
    return rows, positions


def path(tokens, parents, targets, most):
    """The accepted nodes of one sequence."""
    out = [0] if tokens else []
    while out and len(out) < most:
        at = out[-1]
        following = [i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == targets[at]]
        if not following:
            break
        out.append(following[0])
    return out
