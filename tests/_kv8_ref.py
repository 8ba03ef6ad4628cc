"""The 8-bit cache, its attention, its weights and its eviction in 64 bits on the CPU, one element at a time where that is
the definition, from include/kriya_kv8.h alone."""
import math

import torch

BLOCK = 32


def key_at(r, d):
    return d // 16 * 512 + r * 16 + d % 16


def value_at(r, d):
    s, a, h, j = r // 16, r // 8 % 2, r // 4 % 2, r % 4
    return d // 32 * 1024 + h * 512 + d % 32 * 16 + a * 8 + s * 4 + j


def order(d, at):
    """Byte place of every (slot, dim) of a block: int64 [32, d]."""
    r, c = torch.arange(BLOCK)[:, None], torch.arange(d)[None]
    return at(r, c)


def values_of(codes, e4m3):
    return codes.view(torch.float8_e4m3fn).double() if e4m3 else codes.view(torch.int8).double()


def read(cache, n):
    """(k, v) f64 [batch, kv_heads, n, head_dim] of a kv8.Kv8Cache."""
    out = []
    for codes, scale, at in ((cache.k, cache.k_scale, key_at), (cache.v, cache.v_scale, value_at)):
        codes, scale = codes.cpu(), scale.cpu().double()
        x = values_of(codes[..., order(cache.head_dim, at)], cache.format == 1)  # [b, h, blocks, 32, d]
        out.append((x * scale[..., None, None]).flatten(2, 3)[:, :, :n])
    return out


def code(x, e4m3):
    """x f32 [rows <= 32, d] -> (values f64, scale f32), by the definition's two f32 divisions."""
    m = 448.0 if e4m3 else 127.0
    scale = x.abs().max() / m  # (max propagates NaN)
    q = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    q = torch.nan_to_num(q, nan=0.0)
    q = q.clamp(-m, m).to(torch.float8_e4m3fn).double() if e4m3 else q.round().clamp(-m, m).double()
    return q * scale.double(), scale


def rope64(x, cos_sin, positions, layout, inverse=False):
    """x [tokens, heads, d] rotated in 64 bits; tokens past the table unchanged."""
    x, y = x.double(), x.double().clone()
    half = cos_sin.shape[1]
    for t in range(x.shape[0]):
        p = int(positions[t]) & 0xFFFFFFFF
        if p >= cos_sin.shape[0]:
            continue
        for i in range(half):
            c, s = float(cos_sin[p, i, 0]), float(cos_sin[p, i, 1]) * (-1 if inverse else 1)
            a, b = (i, i + half) if layout == 0 else (2 * i, 2 * i + 1)
            y[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            y[t, :, b] = x[t, :, a] * s + x[t, :, b] * c
    return y


def spans(starts, lengths):
    """[(first row, new tokens, length)] of every sequence."""
    n = [int(x) for x in lengths]
    if starts is None:
        return [(b, 1, x) for b, x in enumerate(n)]
    s = [int(x) for x in starts]
    return [(s[b], s[b + 1] - s[b], x) for b, x in enumerate(n)]


def attention(q, k, v, starts, lengths, scale, max_ctx):
    """out, lse, and for error bounds sum p |v| and the largest sum |q k| of a row: q [tokens, heads, d], k, v [batch, kv, slots, d]."""
    tokens, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(tokens, heads, d, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    mass, terms = torch.zeros_like(out), torch.zeros_like(lse)
    weight = torch.zeros(k.shape[0], k.shape[1], max_ctx, dtype=torch.float64)
    q = q.double()
    for b, (t0, m, n) in enumerate(spans(starts, lengths)):
        for i in range(m):
            lim = min(max(n - m + i + 1, 0), max_ctx)
            if lim == 0:
                continue
            for h in range(heads):
                kk, vv = k[b, h // group, :lim], v[b, h // group, :lim]
                x = kk @ q[t0 + i, h] * scale
                p = torch.softmax(x, 0)
                out[t0 + i, h] = p @ vv
                mass[t0 + i, h] = p @ vv.abs()
                lse[t0 + i, h] = torch.logsumexp(x, 0)
                terms[t0 + i, h] = (kk.abs() @ q[t0 + i, h].abs()).max() * abs(scale)
                weight[b, h // group, :lim] += p
    return out, lse, mass, terms, weight


def kept_slots(weight, n, budget, sink, recent):
    """Kept slots of one head, in order, by the definition."""
    if n <= budget:
        return list(range(n))
    w = [float(x) for x in weight[:n]]
    mid = range(sink, n - recent)
    rank = sorted(mid, key=lambda p: (w[p] != w[p], -w[p] if w[p] == w[p] else 0.0, p))
    return sorted(list(range(sink)) + list(range(n - recent, n)) + rank[: budget - sink - recent])
