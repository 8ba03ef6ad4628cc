"""GPU: the 8-bit key/value cache, attention over it, accumulated weights and eviction against 64 bits on the CPU."""
import math

import pytest
import torch

import _kv8_ref as ref

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def kv8(kq):
    from kriya_q4 import kv8

    return kv8


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _starts(counts):
    return _i32([sum(counts[:i]) for i in range(len(counts) + 1)])


def _rand(g, *shape, gain=1.0):
    return (torch.randn(*shape, generator=g) * gain).to(BF)


def _expected(rows, e4m3):
    """Values f64 and scales f32 of bf16 rows [n, heads, d], in blocks of 32: [heads, n, d], [heads, blocks]."""
    vals, scales = [], []
    for h in range(rows.shape[1]):
        v, s = zip(*(ref.code(rows[i: i + 32, h].float(), e4m3) for i in range(0, rows.shape[0], 32)))
        vals.append(torch.cat(v))
        scales.append(torch.stack(s))
    return torch.stack(vals), torch.stack(scales)


def _check_cache(cache, rows_k, rows_v, lengths, e4m3):
    """The cache stands exactly for these bf16 rows ([batch][n, heads, d])."""
    for b, n in enumerate(lengths):
        if not n:
            continue
        k, v = ref.read(cache, n)
        for got, scale, opened, rows in ((k, cache.k_scale, cache.k_open, rows_k), (v, cache.v_scale, cache.v_open, rows_v)):
            want, s = _expected(rows[b][:n], e4m3)
            assert torch.equal(got[b], want)
            assert torch.equal(scale[b, :, : s.shape[1]].cpu(), s)
            last = (n - 1) // 32 * 32
            assert torch.equal(opened[b, :, : n - last].cpu(), rows[b][last:n].transpose(0, 1))


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("d,heads", [(64, 1), (96, 3), (128, 2), (192, 1), (256, 2)])
def test_append_any_way_gives_the_same_cache(kv8, d, heads, e4m3):
    """Token by token, in ragged chunks (with empty ones) or at once: the codes of whole blocks coded at once."""
    g = torch.Generator().manual_seed(d + e4m3)
    lens = [97, 1, 64, 32, 33]
    rk = [_rand(g, n, heads, d) * (1 + 3 * i) for i, n in enumerate(lens)]
    rv = [_rand(g, n, heads, d) for n in lens]
    rk[0][40:] *= 0.01  # block scales far apart
    cut = {"at once": [lens], "one by one": [[1 if i < n else 0 for n in lens] for i in range(97)],
           "chunks": [[31, 0, 1, 32, 2], [2, 1, 63, 0, 29], [64, 0, 0, 0, 2]]}
    for way, steps in cut.items():
        cache = kv8.Kv8Cache(len(lens), heads, d, 100, format=e4m3)
        have = [0] * len(lens)
        for counts in steps:
            k = torch.cat([r[a: a + c] for r, a, c in zip(rk, have, counts)])
            v = torch.cat([r[a: a + c] for r, a, c in zip(rv, have, counts)])
            have = [a + c for a, c in zip(have, counts)]
            kv8.append(cache, k.cuda(), v.cuda(), _i32(have), starts=_starts(counts))
        assert have == lens, way
        _check_cache(cache, rk, rv, lens, e4m3)


def test_append_one_token_each_without_starts_and_strided(kv8):
    g = torch.Generator().manual_seed(1)
    cache, rk, rv = kv8.Kv8Cache(3, 2, 64, 40), [[] for _ in range(3)], [[] for _ in range(3)]
    for step in range(40):
        row = _rand(g, 3, 6 * 64 + 8)  # q, k and v in the row of one projection
        k, v = row[:, 2 * 64: 4 * 64].unflatten(1, (2, 64)), row[:, 4 * 64: 6 * 64].unflatten(1, (2, 64))
        dev = row.cuda()
        kv8.append(cache, dev[:, 128:256].unflatten(1, (2, 64)), dev[:, 256:384].unflatten(1, (2, 64)), _i32([step + 1] * 3))
        for b in range(3):
            rk[b].append(k[b: b + 1])
            rv[b].append(v[b: b + 1])
    _check_cache(cache, [torch.cat(x) for x in rk], [torch.cat(x) for x in rv], [40] * 3, 0)


@pytest.mark.parametrize("rotary,layout", [(128, 0), (64, 1), (36, 0), (32, 0), (50, 1)])
def test_append_rotates_k_and_q(kv8, kq, rotary, layout):
    from kriya_q4 import rope

    g = torch.Generator().manual_seed(rotary)
    counts, d = [3, 0, 40], 128
    t = sum(counts)
    k, v, q = _rand(g, t, 2, d), _rand(g, t, 2, d), _rand(g, t, 6, d)
    table = rope.table(rotary, 60, 1e4)
    pos = torch.randint(0, 60, (t,), generator=g, dtype=I32)
    pos[2] = 60  # past the table: left as it is
    cache = kv8.Kv8Cache(3, 2, d, 64)
    qo = torch.empty_like(q, device="cuda")
    lens = [3, 0, 40]
    kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_starts(counts), q=q.cuda(), q_out=qo, cos_sin=table,
               positions=pos.cuda(), layout=layout)
    # the same rotation as rope.apply, bit for bit, then coded as any rows
    turn = lambda x: rope.apply(x.cuda(), table, pos.cuda(), layout=layout).cpu()  # noqa: E731
    assert torch.equal(qo.cpu(), turn(q))
    rk = turn(k)
    _check_cache(cache, [rk[:3], rk[:0], rk[3:]], [v[:3], v[:0], v[3:]], lens, 0)
    inplace = q.cuda()
    kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_starts(counts), q=inplace, cos_sin=table, positions=pos.cuda(), layout=layout)
    assert torch.equal(inplace.cpu(), qo.cpu())


def test_append_cuts_off_what_does_not_fit(kv8):
    """Slots past max_ctx are not written, lengths below the new tokens keep the last ones, rows of starts past
    the tokens are not read; everything else stays as it was."""
    g = torch.Generator().manual_seed(5)
    k, v = _rand(g, 50, 1, 64), _rand(g, 50, 1, 64)
    cache = kv8.Kv8Cache(4, 1, 64, 40)
    for t in (cache.k, cache.v):
        t.fill_(99)
    cache.k_scale.fill_(5.0)
    cache.v_scale.fill_(5.0)
    # sequence 0: 45 tokens into 40 slots; 1: 2 slots for 3 tokens; 2: nothing new; 3: rows 48 .. 60 of 50
    starts, lens = _i32([0, 45, 48, 48, 61]), _i32([45, 2, 7, 2])
    kv8.append(cache, k.cuda(), v.cuda(), lens, starts=starts)
    rows = lambda x: [x[:40], x[46:48], x[:0], x[48:50]]  # noqa: E731
    _check_cache(cache, rows(k), rows(v), [40, 2, 0, 2], 0)
    assert (cache.k[2] == 99).all() and (cache.v[2] == 99).all() and (cache.k_scale[2] == 5).all()
    assert (cache.k[1, :, 1] == 99).all() and (cache.k_scale[1, :, 1] == 5).all()


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_bad_value_spoils_its_block_only(kv8, bad, e4m3):
    g = torch.Generator().manual_seed(9)
    n, d = 100, 64
    k, v, q = _rand(g, n, 2, d), _rand(g, n, 2, d), _rand(g, n, 4, d)
    k[40, 0, 3] = bad
    v[70, 1, 60] = bad
    cache = kv8.Kv8Cache(1, 2, d, n, format=e4m3)
    kv8.append(cache, k.cuda(), v.cuda(), _i32([n]), starts=_starts([n]))
    dk, dv = (x.cpu() for x in kv8.dequant(cache, _i32([n]), n))
    assert torch.isnan(dk[0, 32:64, 0]).all() and not torch.isnan(dk[0, :32]).any() and not torch.isnan(dk[0, :, 1]).any()
    assert torch.isnan(dv[0, 64:96, 1]).all() and not torch.isnan(dv[0, 96:]).any() and not torch.isnan(dv[0, :, 0]).any()
    out, lse = (x.cpu() for x in kv8.attention(cache, q.cuda(), _i32([n]), starts=_starts([n])))
    # causal: rows before a spoilt block are those of a cache without it, rows that see it are NaN, in its head alone
    assert torch.isfinite(out[:32, :2]).all() and torch.isnan(out[32:, :2]).all() and torch.isnan(lse[32:, :2]).all()
    assert torch.isfinite(out[:64, 2:]).all() and torch.isnan(out[64:, 2:]).all() and torch.isfinite(lse[:, 2:]).all()
    k[40, 0, 3] = v[70, 1, 60] = 0.0
    kv8.append(cache, k.cuda(), v.cuda(), _i32([n]), starts=_starts([n]))
    fine, _ = (x.cpu() for x in kv8.attention(cache, q.cuda(), _i32([n]), starts=_starts([n])))
    assert torch.equal(fine[:32, :2], out[:32, :2]) and torch.equal(fine[:64, 2:], out[:64, 2:])


def test_dequant_ranges(kv8):
    g = torch.Generator().manual_seed(11)
    lens, d = [70, 5, 0], 96
    k, v = _rand(g, 75, 3, d), _rand(g, 75, 3, d)
    cache = kv8.Kv8Cache(3, 3, d, 90)
    kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_starts(lens))
    wk, wv = ref.read(cache, 90)
    for first, count in ((None, 90), (None, 1), ([3, 2, 0], 41), ([69, 5, 89], 6), ([31, -1, 33], 2), ([0, 4, 100], 130)):
        for dt in (torch.float32, BF):
            gk, gv = kv8.dequant(cache, _i32(lens), count, first=None if first is None else _i32(first), dtype=dt)
            for got, want in ((gk, wk), (gv, wv)):
                for b, n in enumerate(lens):
                    f = 0 if first is None else first[b] & 0xFFFFFFFF
                    x = torch.zeros(count, 3, d, dtype=torch.float64)
                    m = max(0, min(count, n - f))
                    x[:m] = want[b, :, f: f + m].transpose(0, 1)
                    assert torch.equal(got[b].cpu(), x.float().to(dt)), (first, count, dt, b)  # code * scale rounded to f32, then to the type


# ---- attention

def _fill(kv8, g, lens, heads, d, e4m3, max_ctx, gain=1.0):
    n = sum(lens)
    k, v = _rand(g, n, heads, d, gain=gain), _rand(g, n, heads, d, gain=gain)
    cache = kv8.Kv8Cache(len(lens), heads, d, max_ctx, format=e4m3)
    for t in (cache.k, cache.v):
        t.fill_(0x55)  # what lies behind the lengths is never used (a valid code in both formats)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(math.nan)
    if n:
        kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_starts(lens))
    return cache


def _check_attention(kv8, cache, q, starts, lengths, scale=None, qd=None, workspace=None):
    d = q.shape[2]
    sc = 1 / math.sqrt(d) if scale is None else scale
    qd = q.cuda() if qd is None else qd
    out, lse = kv8.attention(cache, qd, lengths, starts=starts, scale=scale, workspace=workspace)
    k, v = ref.read(cache, cache.max_ctx)
    want, wl, mass, terms, weight = ref.attention(q, k, v, None if starts is None else starts.cpu(), lengths.cpu(), sc, cache.max_ctx)
    n = float(lengths.max())
    vmax = float(torch.nan_to_num(v).abs().max())
    # scores: D products summed in f32 (and the scales multiplied in); a weight is off by e^that, exp2 by 2 ulp
    off = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -22
    # probabilities in fp16: half a step each, below 2^-14 half of 2^-24 of the largest value; sums of n in f32; output in bf16
    p = 2.0 ** -11 + 2 * off[..., None] + 2 * n * 2.0 ** -24
    tol = 2.0 ** -8 * want.abs() + p * mass + n * 2.0 ** -25 * vmax
    bad = (out.cpu().double() - want).abs() - tol
    assert (bad <= 0).all(), float(bad.max())
    live = wl > -math.inf
    assert torch.equal(lse.cpu() > -math.inf, live)
    lt = off + n * 2.0 ** -24 + 2.0 ** -22 * (1 + wl.abs())
    assert ((lse.cpu().double() - wl).abs()[live] <= lt[live]).all()
    assert (out.cpu()[~live] == 0).all()
    return out, lse, weight, off


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("d,kv,group", [(64, 2, 1), (96, 1, 8), (128, 2, 8), (128, 1, 3), (192, 2, 5), (256, 1, 17), (64, 1, 40)])
def test_attention_one_token_each(kv8, d, kv, group, e4m3):
    g = torch.Generator().manual_seed(d + group)
    lens = [1, 31, 32, 33, 64, 200, 7]
    cache = _fill(kv8, g, lens, kv, d, e4m3, 210)
    _check_attention(kv8, cache, _rand(g, len(lens), kv * group, d, gain=2.0), None, _i32(lens))


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("d,kv,group,counts,lens", [
    (128, 2, 8, [45], [45]), (64, 1, 4, [130, 0, 1, 17], [130, 9, 64, 300]), (96, 3, 1, [33, 2], [40, 200]),
    (256, 1, 5, [70, 1], [100, 65]), (192, 1, 3, [5, 64, 0], [5, 64, 0]), (128, 1, 16, [200], [230])])
def test_attention_ragged_chunks(kv8, d, kv, group, counts, lens, e4m3):
    g = torch.Generator().manual_seed(d + sum(counts))
    cache = _fill(kv8, g, lens, kv, d, e4m3, max(lens) + 3)
    _check_attention(kv8, cache, _rand(g, sum(counts), kv * group, d), _starts(counts), _i32(lens))


@pytest.mark.parametrize("d,kv,group,counts,lens", [
    (64, 2, 4, [40, 0, 9, 1], [3000, 7, 40, 1500]), (128, 1, 3, [60, 100], [1800, 130]), (256, 2, 5, [55, 13, 26], [1999, 1300, 26]),
    (96, 3, 2, [33, 64, 64], [2500, 64, 1025]), (192, 1, 8, [1, 1, 140], [1, 2, 2222]), (128, 8, 1, [200, 3], [900, 2900])])
def test_attention_chunks_whose_tiles_are_shared_out(kv8, d, kv, group, counts, lens):
    """Long contexts under few tiles: workgroups take ends, whole ones and beginnings of tiles, short sequences between long ones."""
    g = torch.Generator().manual_seed(d + group + kv)
    cache = _fill(kv8, g, lens, kv, d, 1 if d == 96 else 0, max(lens) + 3)
    q, lengths = _rand(g, sum(counts), kv * group, d), _i32(lens)
    _check_attention(kv8, cache, q, _starts(counts), lengths)


def test_attention_rows_that_see_nothing_and_cut_lengths(kv8):
    g = torch.Generator().manual_seed(21)
    lens = [40, 3, 0, 33]
    cache = _fill(kv8, g, lens, 2, 64, 0, 40)
    counts = [4, 5, 2, 1]  # sequence 1 has 5 new tokens of 3, sequence 2 2 of none
    out, lse, _, _ = _check_attention(kv8, cache, _rand(g, 12, 4, 64), _starts(counts), _i32(lens))
    assert (lse[4:6].cpu() == -math.inf).all() and (out[9:11] == 0).all()
    # a length beyond max_ctx is cut to it, rows of starts beyond the tokens are not taken
    q = _rand(g, 5, 4, 64).cuda()
    a, la = kv8.attention(cache, q, _i32([60, 3, 0, 33]), starts=_i32([0, 1, 2, 3, 99]))
    b, lb = kv8.attention(cache, q, _i32([40, 3, 0, 33]), starts=_i32([0, 1, 2, 3, 5]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[3:], b[3:]) and torch.equal(la[1], lb[1])


def test_lengths_of_any_size_see_the_whole_cache_and_no_more(kv8):
    """Lengths up to 2^32 - 1, the largest (-1 as int32): every slot there is, as for a length of max_ctx and all its tokens old."""
    g = torch.Generator().manual_seed(29)
    cache = _fill(kv8, g, [100, 100], 2, 64, 0, 100)
    for counts in ([1, 1], [70, 3]):
        starts, m = _starts(counts), sum(counts)
        q = _rand(g, m, 4, 64).cuda()
        lens = _i32([-1, 100 + counts[1]])
        out, lse = kv8.attention(cache, q, lens, starts=starts)
        each, each_lse = [], []
        for t in range(m):  # each row by itself, at a length that sees all
            b = int(t >= counts[0])
            c = kv8.Kv8Cache.wrap(*(x[b:b + 1] for x in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_open, cache.v_open)), 100)
            o, l = kv8.attention(c, q[t:t + 1], _i32([100]))
            each.append(o)
            each_lse.append(l)
        # fp16 probabilities in another grouping: 2^-11 of values below 6, and bf16's half step twice
        assert (out.float() - torch.cat(each).float()).abs().max() <= 2 * (2.0 ** -11 + 2.0 ** -8) * 6
        assert (lse - torch.cat(each_lse)).abs().max() <= 1e-5
        w = kv8.accumulate_weight(cache, q, lse, lens, torch.zeros(2, 2, 100, device="cuda"), starts=starts)
        got = w.sum(-1)  # every row's weights add up to one
        assert (got - torch.tensor(counts, device="cuda")[:, None] * 2.0).abs().max() <= 1e-4 * max(counts)


@pytest.mark.parametrize("gain", [1e-30, 1e-6, 1e3, 1e30])
def test_attention_range_of_values(kv8, gain):
    """bf16 range: q and k of any size whose scores stay in f32, values of any size, blocks of values far apart."""
    g = torch.Generator().manual_seed(4)
    n, d = 150, 64
    k, v = _rand(g, n, 1, d), _rand(g, n, 1, d)
    v[40:] *= 2.0 ** 20
    v[100:] *= 2.0 ** -30
    v = (v.float() * gain).to(BF)
    q = (_rand(g, 3, 2, d).float() / gain).to(BF)
    k = (k.float() * gain).to(BF)
    cache = kv8.Kv8Cache(1, 1, d, n)
    kv8.append(cache, k.cuda(), v.cuda(), _i32([n]), starts=_starts([n]))
    _check_attention(kv8, cache, q, _starts([3]), _i32([n]))
    q = (_rand(g, 40, 2, d).float() / gain).to(BF)  # as a chunk of many rows
    _check_attention(kv8, cache, q, _starts([40]), _i32([n]))


@pytest.mark.parametrize("m", [1, 60])
def test_attention_over_values_near_the_smallest(kv8, m):
    """Values whose scales are subnormal floats, blocks of zeros among them: within the codes' own steps of the exact result."""
    g = torch.Generator().manual_seed(14)
    n, d = 130, 64
    k, v = _rand(g, n, 1, d), (_rand(g, n, 1, d).float() * 2.0 ** -122).to(BF)
    v[32:64] = 0.0
    cache = kv8.Kv8Cache(1, 1, d, n)
    kv8.append(cache, k.cuda(), v.cuda(), _i32([n]), starts=_starts([n]))
    q = _rand(g, m, 2, d)
    out, _ = kv8.attention(cache, q.cuda(), _i32([n]), starts=_starts([m]))
    _, vv = ref.read(cache, n)
    want, _, mass, _, _ = ref.attention(q, *ref.read(cache, n), torch.tensor([0, m]), [n], 1 / 8, n)
    # P and V relative to 2^-126 in fp16 (P's steps below 2^-14 are 2^-24, times codes up to 127), outputs in bf16 (subnormal step 2^-133)
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -10 * mass + n * 127 * 2.0 ** -25 * 2.0 ** -126 + 2.0 ** -133
    assert (((out.cpu().double() - want).abs() - tol) <= 0).all() and float(want.abs().max()) > 0


def test_attention_strided_queries_peaked_and_infinite_rows(kv8):
    g = torch.Generator().manual_seed(8)
    lens = [90, 64]
    cache = _fill(kv8, g, lens, 2, 128, 0, 100)
    buf = _rand(g, 2, 12 * 128, gain=30.0)  # peaked: scores of hundreds
    view = lambda t: t[:, 4 * 128: 8 * 128].unflatten(1, (4, 128))  # noqa: E731
    dev = buf.cuda()
    out, lse, _, _ = _check_attention(kv8, cache, view(buf), None, _i32(lens), qd=view(dev))
    dev[0, 4 * 128 + 5] = math.inf  # one head of one token
    o2, l2 = kv8.attention(cache, view(dev), _i32(lens))
    assert torch.isnan(o2[0, 0]).all() and torch.isnan(l2[0, 0])
    assert torch.equal(o2[0, 1:], out[0, 1:]) and torch.equal(o2[1], out[1]) and torch.equal(l2[1], lse[1])


@pytest.mark.parametrize("scale", [-0.25, 0.0, 1.5])
@pytest.mark.parametrize("m", [1, 50])
def test_attention_and_weights_at_any_scale(kv8, scale, m):
    g = torch.Generator().manual_seed(19)
    n, d = 200, 64
    cache = _fill(kv8, g, [n], 2, d, 0, n)
    q, starts, lens = _rand(g, m, 4, d), _starts([m]), _i32([n])
    out, lse, want, off = _check_attention(kv8, cache, q, starts, lens, scale=scale)
    w = kv8.accumulate_weight(cache, q.cuda(), lse, lens, torch.zeros(1, 2, n, device="cuda"), starts=starts, scale=scale)
    tol = (4 * float(off.max()) + (n + 2 * m) * 2.0 ** -24 + 2.0 ** -20) * want + 1e-30
    assert ((w.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("gain", [1e-30, 1e30])
@pytest.mark.parametrize("m", [1, 50])
def test_accumulated_weights_range_of_values(kv8, gain, m):
    """Keys near the ends of f32 against queries near the other: scores of ordinary size."""
    g = torch.Generator().manual_seed(31)
    n, d = 300, 96
    cache = _fill(kv8, g, [n], 2, d, 0, n, gain=gain)
    q, starts, lens = (_rand(g, m, 4, d).float() / gain).to(BF), _starts([m]), _i32([n])
    out, lse, want, off = _check_attention(kv8, cache, q, starts, lens)
    w = kv8.accumulate_weight(cache, q.cuda(), lse, lens, torch.zeros(1, 2, n, device="cuda"), starts=starts)
    tol = (4 * float(off.max()) + (n + 2 * m) * 2.0 ** -24 + 2.0 ** -20) * want + 1e-30
    assert ((w.cpu().double() - want).abs() <= tol).all()


def test_calls_on_another_stream_with_workspaces_of_their_own(kv8):
    """Calls on a side stream whose workspaces are freed as soon as they return, while the current stream allocates and fills."""
    g = torch.Generator().manual_seed(23)
    cache = _fill(kv8, g, [3000, 2000], 2, 64, 0, 3000)
    q, lens = _rand(g, 400, 8, 64).cuda(), _i32([3000, 2000])
    starts = _starts([300, 100])
    own, lse = kv8.attention(cache, q, lens, starts=starts)
    weight = kv8.accumulate_weight(cache, q, lse, lens, torch.zeros(2, 2, 3000, device="cuda"), starts=starts)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        got = []
        for _ in range(4):
            w = torch.zeros(2, 2, 3000, device="cuda")
            side.wait_stream(torch.cuda.current_stream())
            a = kv8.attention(cache, q, lens, starts=starts, stream=stream)
            kv8.accumulate_weight(cache, q, lse, lens, w, starts=starts, stream=stream)
            torch.full((8 << 20,), 255, dtype=torch.uint8, device="cuda")
            got.append((a, w))
        side.synchronize()
        for (o, l), w in got:
            assert torch.equal(o, own) and torch.equal(l, lse) and torch.equal(w, weight)


@pytest.mark.parametrize("counts,lens", [([1, 1], [900, 40]), ([1, 0], [40, 9]), ([90, 30], [70, 2600]), ([60, 50], [200, 300])])
def test_rows_behind_the_last_sequence_and_no_lse(kv8, kq, counts, lens):
    """Seven rows more than the sequences have: their results stay as they were.  Without lse: the same output."""
    g = torch.Generator().manual_seed(37)
    ctx = max(lens) + max(counts)
    cache = _fill(kv8, g, lens, 2, 64, 0, ctx)
    n, starts, lengths = sum(counts), _starts(counts), _i32(lens)
    q = _rand(g, n + 7, 8, 64).cuda()
    out, lse = torch.full_like(q, 3.0), torch.full((n + 7, 8), 5.0, device="cuda")
    kv8.attention(cache, q, lengths, starts=starts, out=out, lse=lse)
    assert (out[n:] == 3.0).all() and (lse[n:] == 5.0).all()
    want, want_lse = kv8.attention(cache, q[:n], lengths, starts=starts)
    sees = want_lse > -math.inf  # (a row of a sequence with more new tokens than tokens may see none)
    assert (out[:n].float() - want.float()).abs().max() <= 2 * (2.0 ** -11 + 2.0 ** -8) * 6
    assert torch.equal(lse[:n] > -math.inf, sees) and (lse[:n] - want_lse)[sees].abs().max() <= 1e-5
    bare, ws = torch.full_like(q, 3.0), kv8.attention_workspace(cache, 8, n + 7)
    kq._check(kq.lib().kr_kv8_attention(cache.desc, q.data_ptr(), 512, 8, n + 7, starts.data_ptr(), lengths.data_ptr(), 0.125,
                                        bare.data_ptr(), None, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(bare, out)
    weight = kv8.accumulate_weight(cache, q, lse, lengths, torch.zeros(2, 2, ctx, device="cuda"), starts=starts)
    live = torch.tensor([min(c, k) for c, k in zip(counts, lens)], device="cuda")
    assert (weight.sum(-1) - live[:, None] * 4.0).abs().max() <= 1e-4 * max(counts) * 4
    rows = torch.full((n + 7, 2, 64), float("nan"), dtype=BF, device="cuda")
    rows[:n] = 1.0
    before = cache.k.clone(), cache.v_scale.clone(), cache.k_open.clone()
    two = kv8.Kv8Cache.wrap(before[0], cache.v.clone(), cache.k_scale.clone(), before[1], before[2], cache.v_open.clone(), ctx)
    longer = [a + b for a, b in zip(lens, counts)]
    kv8.append(cache, rows, rows, _i32(longer), starts=starts)
    kv8.append(two, rows[:n].contiguous(), rows[:n].contiguous(), _i32(longer), starts=starts)
    for x, y in zip(ref.read(cache, ctx), ref.read(two, ctx)):  # (slots behind the lengths hold what they held)
        assert all(torch.equal(x[b, :, :k], y[b, :, :k]) for b, k in enumerate(longer))


def test_attention_takes_back_tokens_of_the_last_block(kv8):
    g = torch.Generator().manual_seed(6)
    cache = _fill(kv8, g, [60], 1, 64, 0, 64)
    _check_attention(kv8, cache, _rand(g, 1, 2, 64), None, _i32([50]))
    k, v = _rand(g, 1, 1, 64), _rand(g, 1, 1, 64)
    kv8.append(cache, k.cuda(), v.cuda(), _i32([51]))
    assert torch.equal(cache.k_open[0, 0, 18].cpu(), k[0, 0])
    _check_attention(kv8, cache, _rand(g, 1, 2, 64), None, _i32([51]))


@pytest.mark.parametrize("batch", [63, 64, 65, 130])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_sequences(kv8, batch, ragged):
    """Batches around and past a wave's lanes, with empty sequences in them: appended, attended, weighted."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 60, (batch,), generator=g).tolist()
    counts = [min(n, c) for n, c in zip(lens, torch.randint(0, 9, (batch,), generator=g).tolist())]
    lens[-1], counts[-1] = 300, 200 if ragged else 1
    if ragged:
        lens[0] = counts[0] = 0
    else:
        counts = [1] * batch
    cache = _fill(kv8, g, lens, 1, 64, 0, 310)
    starts = _starts(counts) if ragged else None
    q = _rand(g, sum(counts), 3, 64)
    out, lse, want, off = _check_attention(kv8, cache, q, starts, _i32(lens))
    w = torch.zeros(batch, 1, 310, device="cuda")
    kv8.accumulate_weight(cache, q.cuda(), lse, _i32(lens), w, starts=starts)
    want = want.clone()
    tol = (4 * float(off.max()) + 900 * 2.0 ** -24 + 2.0 ** -20) * want + 1e-30
    assert ((w.cpu().double() - want).abs() <= tol).all()


def test_calls_that_share_a_workspace_and_replays(kv8):
    """One workspace under calls of many shapes back to back (decoding in parts, chunks in parts, whole prompts), eager and
    captured, gives each call's own bits; 24 rounds."""
    g = torch.Generator().manual_seed(33)
    calls = []
    for lens, counts, kv, group, d in (([3000] * 3 + [1, 2500], None, 2, 4, 64), ([4000], None, 1, 3, 64), ([2000, 3000], [40, 3], 1, 8, 64),
                                       ([700] * 9, None, 8, 1, 64), ([6000], None, 1, 16, 128), ([500, 900] * 20, None, 2, 2, 96)):
        cache = _fill(kv8, g, lens, kv, d, 0, max(lens))
        starts = None if counts is None else _starts(counts)
        q = _rand(g, len(lens) if counts is None else sum(counts), kv * group, d).cuda()
        calls.append((cache, q, _i32(lens), starts))
    own = [kv8.attention(*c[:3], starts=c[3]) for c in calls]
    ws = max((kv8.attention_workspace(c[0], c[1].shape[1], c[1].shape[0]) for c in calls), key=lambda t: t.numel()).fill_(255)
    outs = [(torch.empty_like(o), torch.empty_like(l)) for o, l in own]

    def all_calls():
        for (cache, q, n, st), (o, l) in zip(calls, outs):
            kv8.attention(cache, q, n, starts=st, out=o, lse=l, workspace=ws)
    all_calls()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            all_calls()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(24):
        for o, l in outs:
            o.zero_()
            l.zero_()
        if i % 2:
            graph.replay()
        else:
            all_calls()
        if i % 5 == 0:
            torch.cuda.synchronize()
        for (o, l), (wo, wl) in zip(outs, own):
            assert torch.equal(o, wo) and torch.equal(l, wl), i


def test_attention_across_more_than_4_gib(kv8):
    """Offsets past 32 bits: the last sequence of a cache whose keys alone are more than 4 GiB."""
    g = torch.Generator().manual_seed(2)
    b, h, d, ctx = 34, 8, 128, 1 << 17
    cache = kv8.Kv8Cache(b, h, d, ctx)
    assert cache.k.numel() > 1 << 32
    n = 100
    lens = [0] * (b - 1) + [n]
    k, v = _rand(g, n, h, d), _rand(g, n, h, d)
    kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_i32([0] * b + [n]))
    small = kv8.Kv8Cache(1, h, d, n)
    kv8.append(small, k.cuda(), v.cuda(), _i32([n]), starts=_i32([0, n]))
    q = _rand(g, 2, 2 * h, d).cuda()
    out, lse = kv8.attention(cache, q, _i32(lens), starts=_i32([0] * b + [2]))
    o1, l1 = kv8.attention(small, q, _i32([n]), starts=_i32([0, 2]))
    assert (out.float() - o1.float()).abs().max() <= 2.0 ** -7 and (lse - l1).abs().max() <= 2.0 ** -18
    assert all(torch.equal(x[-1, :n], y[0]) for x, y in zip(kv8.dequant(cache, _i32(lens), n), kv8.dequant(small, _i32([n]), n)))
    w, w1 = torch.zeros(b, h, ctx, device="cuda"), torch.zeros(1, h, n, device="cuda")
    kv8.accumulate_weight(cache, q, l1, _i32(lens), w, starts=_i32([0] * b + [2]))
    kv8.accumulate_weight(small, q, l1, _i32([n]), w1, starts=_i32([0, 2]))
    assert torch.equal(w[-1, :, :n], w1[0])


def test_a_very_long_context(kv8):
    """One sequence of 2^20 + 7 slots, decoded and as a chunk: a key far down draws all the attention, and uniform weights average."""
    n, d = (1 << 20) + 7, 64
    k, v = torch.zeros(n, 1, d, dtype=BF, device="cuda"), torch.zeros(n, 1, d, dtype=BF, device="cuda")
    v[:, 0, 0] = 1.0
    v[1 << 19:, 0, 1] = 1.0
    k[n - 40, 0, 2] = 64.0
    v[n - 40, 0, 3] = -1.0
    cache = kv8.Kv8Cache(1, 1, d, n)
    kv8.append(cache, k, v, _i32([n]), starts=_i32([0, n]))
    for m in (1, 70):
        q = torch.zeros(m, 2, d, dtype=BF, device="cuda")
        q[:, 1, 2] = 16.0
        out, lse = kv8.attention(cache, q, _i32([n]), starts=_i32([0, m]), scale=1.0)
        o, ls = out.cpu().double(), lse.cpu().double()
        for i in range(m):
            seen = n - m + i + 1
            assert abs(ls[i, 0] - math.log(seen)) <= 1e-5 * 14
            assert abs(o[i, 0, 0] - 1.0) <= 2.0 ** -8 and abs(o[i, 0, 1] - (seen - (1 << 19)) / seen) <= 2.0 ** -8
            if seen > n - 40:
                assert abs(o[i, 1, 3] + 1.0) <= 2.0 ** -7 and abs(ls[i, 1] - 1024.0) <= 1e-3


# ---- accumulated weights and eviction

@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("d,kv,group,counts,lens", [
    (128, 2, 8, None, [1, 33, 200]), (64, 1, 3, [40, 0, 1], [40, 70, 64]), (256, 1, 2, [5, 100], [300, 100]),
    (96, 2, 20, None, [64, 5, 31]), (192, 1, 1, [70], [75])])
def test_accumulated_weights(kv8, d, kv, group, counts, lens, e4m3):
    g = torch.Generator().manual_seed(d)
    ctx = max(lens) + 9
    cache = _fill(kv8, g, lens, kv, d, e4m3, ctx)
    t = len(lens) if counts is None else sum(counts)
    starts, lengths = None if counts is None else _starts(counts), _i32(lens)
    q = _rand(g, t, kv * group, d)
    out, lse, want, off = _check_attention(kv8, cache, q, starts, lengths)
    had = torch.rand(len(lens), kv, ctx, generator=g)
    w = had.clone().cuda()
    new = [1] * len(lens) if counts is None else counts
    for b, (m, n) in enumerate(zip(new, lens)):
        w[b, :, n - m: n] = math.nan  # new slots start at zero whatever was there
    before = w.cpu().clone()
    kv8.accumulate_weight(cache, q.cuda(), lse, lengths, w, starts=starts, decay=0.75)
    for b, (m, n) in enumerate(zip(new, lens)):
        x = torch.zeros(kv, n, dtype=torch.float64)
        x[:, : n - m] = 0.75 * had[b, :, : n - m].double()
        x += want[b, :, :n]
        # the scores' and lse's errors, exp2, and a sum of m * group terms in f32
        tol = (4 * float(off.max()) + (n + m * group) * 2.0 ** -24 + 2.0 ** -20) * x + 1e-30
        assert ((w[b, :, :n].cpu().double() - x).abs() <= tol).all()
        assert torch.equal(w[b, :, n:].cpu(), before[b, :, n:])


def _check_evicted(cache, to, lens, weight, kept, to_lengths, to_weight, budget, sink, recent, raw_k, raw_v, before):
    e4m3 = cache.format == 1
    old, new = ref.read(cache, cache.max_ctx), ref.read(to, to.max_ctx)
    for b, n in enumerate(lens):
        left = min(n, budget)
        assert int(to_lengths[b]) == left
        for h in range(cache.kv_heads):
            slots = ref.kept_slots(weight[b, h], n, budget, sink, recent)
            assert kept[b, h, :left].tolist() == slots
            assert torch.equal(to_weight[b, h, :left].nan_to_num(-1), weight[b, h, slots].nan_to_num(-1))
            assert torch.equal(to_weight[b, h, left:], before[b, h, left:])
            for side, (got, held, raw, scale, opened, src) in enumerate((
                    (new[0], old[0], raw_k, to.k_scale, to.k_open, cache.k_scale), (new[1], old[1], raw_v, to.v_scale, to.v_open, cache.v_scale))):
                for i in range(0, left, 32):
                    rows = slots[i: i + 32]
                    final = i + 32 >= left
                    x = held[b, h, rows]
                    if n <= budget or (not final and rows[-1] == i + 31):
                        assert torch.equal(got[b, h, i: i + len(rows)], x)
                        assert scale[b, h, i // 32].cpu() == src[b, h, i // 32].cpu()
                        continue
                    tail = (n - 1) // 32 * 32
                    x = x.float()  # code * scale in f32
                    for r, p in enumerate(rows):
                        if p >= tail:
                            x[r] = raw[b][p, h].float()
                    if final:
                        x = x.to(BF).float()
                        assert torch.equal(opened[b, h, : len(rows)].cpu().float(), x)
                    y, s = ref.code(x, e4m3)
                    assert torch.equal(got[b, h, i: i + len(rows)], y) and scale[b, h, i // 32].cpu() == s


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("d,heads,lens,budget,sink,recent", [
    (64, 2, [100, 70, 30, 0], 70, 4, 20), (128, 1, [300], 33, 0, 0), (96, 3, [65, 64, 40], 40, 40, 0), (192, 1, [129, 96], 96, 0, 96),
    (256, 2, [200, 97], 96, 32, 31), (64, 1, [2500, 2100], 1, 0, 0), (64, 1, [2500, 1200], 1100, 1, 1000)])
def test_evict(kv8, d, heads, lens, budget, sink, recent, e4m3):
    g = torch.Generator().manual_seed(budget)
    ctx = max(lens) + 5
    rk, rv = [_rand(g, n, heads, d) for n in lens], [_rand(g, n, heads, d) for n in lens]
    cache = kv8.Kv8Cache(len(lens), heads, d, ctx, format=e4m3)
    kv8.append(cache, torch.cat(rk).cuda(), torch.cat(rv).cuda(), _i32(lens), starts=_starts(lens))
    weight = (torch.rand(len(lens), heads, ctx, generator=g) * 8).round() / 8  # many ties
    weight[:, :, ::7] = 0.0
    weight[:, 0, 3::11] = -0.0
    weight[:, :, 5::13] = math.nan
    weight[:, 0, 6::17] = math.inf
    weight[:, -1, 8::19] = -math.inf
    to = kv8.Kv8Cache(len(lens), heads, d, budget + 3, format=e4m3)
    before = torch.rand(len(lens), heads, budget + 3, generator=g)
    to_weight = before.clone().cuda()
    kept, to_lengths = kv8.evict(cache, _i32(lens), weight.cuda(), budget, sink, recent, to, to_weight)
    _check_evicted(cache, to, lens, weight, kept.cpu(), to_lengths.cpu(), to_weight.cpu(), budget, sink, recent, rk, rv, before)


@pytest.mark.parametrize("n,budget", [(5000, 1777), (16384, 9000), (16385, 400), (40000, 39990)])
def test_evict_many_equal_weights_and_order_of_floats(kv8, n, budget):
    g = torch.Generator().manual_seed(77)
    cache = _fill(kv8, g, [n, n], 1, 64, 0, n)
    weight = torch.zeros(2, 1, n)
    weight[1, 0] = torch.randn(n, generator=g) * torch.exp(20 * torch.randn(n, generator=g))  # every exponent, both signs
    to = kv8.Kv8Cache(2, 1, 64, budget)
    kept, _ = kv8.evict(cache, _i32([n, n]), weight.cuda(), budget, 3, min(70, budget - 3), to, torch.empty(2, 1, budget, device="cuda"))
    for b in range(2):
        assert kept[b, 0].tolist() == ref.kept_slots(weight[b, 0], n, budget, 3, min(70, budget - 3))


def test_binding_refuses(kv8):
    cache = kv8.Kv8Cache(2, 2, 64, 40)
    x = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    n = _i32([1, 1])
    with pytest.raises(ValueError):
        kv8.append(cache, x.float(), x, n)
    with pytest.raises(ValueError):
        kv8.append(cache, x, x[:1], n)
    with pytest.raises(ValueError):
        kv8.append(cache, x, x, n.long())
    with pytest.raises(ValueError):
        kv8.append(cache, x, x, n, starts=n)
    with pytest.raises(ValueError):
        kv8.append(cache, x, x, n, cos_sin=torch.zeros(3, 32, 2, device="cuda"))
    with pytest.raises(RuntimeError):
        kv8.append(cache, x, x, n, q=x)
    with pytest.raises(ValueError):
        kv8.attention(cache, torch.zeros(2, 2, 128, dtype=BF, device="cuda"), n)
    with pytest.raises(RuntimeError):
        kv8.attention(cache, torch.zeros(2, 3, 64, dtype=BF, device="cuda"), n)
    with pytest.raises(RuntimeError):
        kv8.attention(cache, torch.zeros(3, 2, 64, dtype=BF, device="cuda"), n)
    with pytest.raises(ValueError):
        kv8.accumulate_weight(cache, x, torch.zeros(2, 2, device="cuda"), n, torch.zeros(2, 2, 41, device="cuda"))
    with pytest.raises(RuntimeError):
        kv8.evict(cache, n, torch.zeros(2, 2, 40, device="cuda"), 41, 0, 0, kv8.Kv8Cache(2, 2, 64, 40), torch.zeros(2, 2, 40, device="cuda"))
    with pytest.raises(RuntimeError):
        kv8.Kv8Cache(1, 1, 80, 40) and kv8.append(kv8.Kv8Cache(1, 1, 80, 40), torch.zeros(1, 1, 80, dtype=BF, device="cuda"),
                                                  torch.zeros(1, 1, 80, dtype=BF, device="cuda"), _i32([1]))
