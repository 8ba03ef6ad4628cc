"""GPU: the paged key/value cache and the attention over it against 64 bits on the CPU."""
import math
import random

import pytest
import torch

import _paged_ref as ref
from _kv8_ref import rope64

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def paged(kq):
    from kriya_q4 import paged

    return paged


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _starts(counts):
    return _i32([sum(counts[:i]) for i in range(len(counts) + 1)])


def _rand(g, *shape, gain=1.0):
    return (torch.randn(*shape, generator=g) * gain).to(BF)


COLUMNS = 1  # of a table behind its longest sequence's pages


@pytest.fixture(params=[1, 6000], ids=["narrow", "wide"])
def table_of(request):
    """The launch is planned by what a table could hold: in a wide one, many rows take tiles of 128 and may be split; in a narrow one
    short contexts take tiles of 16, or whole ones of 128."""
    global COLUMNS
    COLUMNS = request.param
    yield
    COLUMNS = 1


wide_and_narrow = pytest.mark.usefixtures("table_of")


def _table(lens, page, seed=0, spare=2):
    """Scattered pages for sequences of these lengths: (table rows, pages of the pool)."""
    each = [-(-n // page) for n in lens]
    order = list(range(sum(each) + spare))
    random.Random(seed).shuffle(order)
    rows, at = [], 0
    for n in each:
        rows.append(order[at: at + n] + [-1] * (max(each) - n + COLUMNS))
        at += n
    return rows, len(order)


class Filled:
    """A pool of random bits (NaN among them) with the tokens of sequences of these lengths in its pages, and the same in 64 bits."""

    def __init__(self, paged, lens, kv, d, page, seed=1, gain=1.0, layers=1, layer=0, spare=2):
        self.lens, self.kv, self.d, self.page, self.layer = lens, kv, d, page, layer
        g = torch.Generator().manual_seed(seed)
        rows, pages = _table(lens, page, seed, spare)
        if not rows[0]:
            rows = [r + [-1] for r in rows]
        junk = torch.randint(-(1 << 15), 1 << 15, (2, layers, pages, kv, page // 16, 16 * d), generator=g, dtype=torch.int16)
        self.cache = paged.PagedCache.wrap(*junk.cuda().view(BF).unbind(0))
        self.rows = rows
        self.table, self.lengths = _i32(rows), _i32(lens)
        self.k, self.v = (_rand(g, sum(lens), kv, d, gain=x) for x in (1.0, gain))
        if sum(lens):
            paged.append(self.cache, paged.Step(self.table, self.lengths, _starts(lens)), self.k.cuda(), self.v.cuda(), layer)

    def sequence(self, b):
        """k, v f64 [kv, n, d]."""
        t0, n = sum(self.lens[:b]), self.lens[b]
        return [x[t0: t0 + n].transpose(0, 1).double() for x in (self.k, self.v)]

    def pages(self, b):
        return [p if 0 <= p < self.cache.pages else None for p in self.rows[b]]


def _check(f, paged, q, counts, scale=None, mask=None, words=None, workspace=None, p_half=2.0 ** -8, gpu_q=None, lens=None):
    """attention over f for q [tokens, heads, d] on the CPU; returns (out, lse) on the CPU."""
    lens = f.lens if lens is None else lens
    starts = None if counts is None else _starts(counts)
    step = paged.Step(f.table, f.lengths, starts)
    gm = None
    if mask is not None:
        gm = torch.tensor([[x - (1 << 32) if x >> 31 else x for x in r] for r in mask], dtype=I32, device="cuda")
    out, lse = paged.attention(f.cache, step, q.cuda() if gpu_q is None else gpu_q, f.layer, mask=gm, scale=scale, workspace=workspace)
    out, lse = out.cpu(), lse.cpu()
    d = f.d
    scale = 1 / math.sqrt(d) if scale is None else scale
    for b, (t0, m, n) in enumerate(ref.spans(None if starts is None else starts.tolist(), lens)):
        if not m:
            continue
        k, v = f.sequence(b)
        seen = ref.sees(m, n, k.shape[1], None if mask is None else mask[t0: t0 + m])
        want, wl, mass, terms = ref.attention(q[t0: t0 + m], k, v, seen, scale)
        # a score's error: d products summed in f32 and the factor of the exponent; a weight's: two scores, the sums over n slots,
        # and the rounding of a probability before the second product; the result's rounding to bf16
        off = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -22
        p = p_half + 2 * off[..., None] + 4 * n * 2.0 ** -24
        tol = 2.0 ** -8 * (1 + p) * want.abs() + (1 + 2.0 ** -8) * p * mass
        bad = (out[t0: t0 + m].double() - want).abs() - tol
        assert (bad <= 0).all(), (b, float(bad.max()))
        none = torch.isinf(wl)
        assert torch.equal(torch.isneginf(lse[t0: t0 + m]), none)
        lt = off + n * 2.0 ** -24 + 2.0 ** -22 * (1 + wl.abs())
        assert (none | ((lse[t0: t0 + m].double() - wl).abs() <= lt)).all()
    return out, lse


# ---- appending

@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d,kv", [(64, 1), (96, 3), (128, 2), (192, 1), (256, 2)])
def test_append_any_way_gives_the_same_pages(paged, d, kv, page):
    """At once, in ragged chunks or token by token, into layer 1: the same bits, those of the definition, and no other slot touched."""
    lens = [77, 0, 1, 160]
    f = Filled(paged, lens, kv, d, page, seed=d, layers=2, layer=1)
    for b, n in enumerate(lens):
        for name, pool, rows in (("k", f.cache.k, f.k), ("v", f.cache.v, f.v)):
            got = ref.slots_of(pool[1], name, f.pages(b), page)[:, :n]
            t0 = sum(lens[:b])
            assert torch.equal(got, rows[t0: t0 + n].transpose(0, 1).double())
    h = torch.Generator().manual_seed(d)
    junk = torch.randint(-(1 << 15), 1 << 15, (2,) + tuple(f.cache.k.shape), generator=h, dtype=torch.int16)
    other = paged.PagedCache.wrap(*junk.cuda().view(BF).unbind(0))
    assert torch.equal(other.k[0].view(torch.int16), f.cache.k[0].view(torch.int16))  # the other layer is as it was
    done, chunks = [0] * 4, [[5, 0, 1, 16], [1, 0, 0, 1], [60, 0, 0, 100]] + [[1 if x < n else 0 for x, n in zip([66 + i, 0, 1, 117 + i], lens)] for i in range(43)]
    for chunk in chunks:
        rows = [sum(lens[:b]) + done[b] + i for b in range(4) for i in range(chunk[b])]
        done = [x + c for x, c in zip(done, chunk)]
        if rows:
            paged.append(other, paged.Step(f.table, _i32(done), _starts(chunk)), f.k[rows].cuda(), f.v[rows].cuda(), 1)
    assert done == lens
    for a, b in ((other.k, f.cache.k), (other.v, f.cache.v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    k, v = paged.read(other, paged.Step(f.table, f.lengths), 170, 1, first=_i32([3, 0, 0, 9]), dtype=torch.float32)
    for b, x in enumerate([3, 0, 0, 9]):
        kk, vv = f.sequence(b)
        left = max(0, min(170, lens[b] - x))
        for got, want in ((k, kk), (v, vv)):
            assert torch.equal(got[b, :left].cpu().double(), want[:, x: x + left].transpose(0, 1)) and not got[b, left:].any()


@pytest.mark.parametrize("rotary,layout", [(128, 0), (64, 1), (36, 0), (50, 1), (0, 0)])
@pytest.mark.parametrize("norms", ["none", "both", "k", "q"])
def test_append_normalises_and_rotates(paged, kq, rotary, layout, norms):
    from kriya_q4 import rope

    d, kv, qh, counts, lens = 128, 2, 20, [5, 0, 30], [40, 7, 30]
    if not rotary and norms == "none":
        return
    g = torch.Generator().manual_seed(rotary + layout)
    rows, pages = _table(lens, 16, 3)
    cache = paged.PagedCache(1, pages, 16, kv, d)
    cache.k.zero_()
    cache.v.zero_()
    t = sum(counts)
    wide = _rand(g, t, kv + kv + qh + 1, d).cuda()  # q, k, v in the rows of a fused projection
    k, v, q = wide[:, :kv], wide[:, kv: 2 * kv], wide[:, 2 * kv: 2 * kv + qh]
    before = wide.cpu()
    qn, kn = ((1 + 0.1 * torch.randn(d, generator=g)).to(BF) for _ in "qk")
    qn, kn = (qn if norms in ("both", "q") else None), (kn if norms in ("both", "k") else None)
    pos = torch.randint(0, 60, (t,), generator=g, dtype=I32)
    pos[3] = 77  # past the table: not rotated
    cs = rope.table(rotary, 60, 1e4) if rotary else None
    paged.append(cache, paged.Step(_i32(rows), _i32(lens), _starts(counts)), k, v, q=q, cos_sin=cs, positions=pos.cuda() if rotary else None,
                 layout=layout, q_norm=None if qn is None else qn.cuda(), k_norm=None if kn is None else kn.cuda(), eps=1e-5)
    got_k, got_v = paged.read(cache, paged.Step(_i32(rows), _i32(lens)), 40, dtype=torch.float32)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()
        return rope64(x, cs.cpu(), pos, layout) if rotary else x
    # one rounding to bf16, and a few in f32 before it (two products of a pair: as large as the pair)
    near = lambda a, b, x: ((a.double() - b).abs() <= 2.0 ** -8 * (1 + 2.0 ** -16) * b.abs() + 2.0 ** -20 * x.abs().amax(-1, keepdim=True)).all()  # noqa: E731
    want = turned(before[:, 2 * kv: 2 * kv + qh], qn)
    assert near(q.cpu(), want, want)
    want, t0 = turned(before[:, :kv], kn), 0
    for b, (m, n) in enumerate(zip(counts, lens)):
        assert near(got_k[b, n - m: n].cpu(), want[t0: t0 + m], want[t0: t0 + m])
        assert torch.equal(got_v[b, n - m: n].cpu(), before[t0: t0 + m, kv: 2 * kv].float())
        assert not got_k[b, : n - m].any() and not got_v[b, : n - m].any()
        t0 += m
    assert torch.equal(wide[:, :2 * kv].cpu(), before[:, :2 * kv]) and torch.equal(wide[:, -1].cpu(), before[:, -1])


def test_append_without_starts_cuts_off_and_skips_missing_pages(paged):
    """One token each; a length past the table, one below its new tokens, and a slot whose page is none: nothing else is written."""
    d, kv = 64, 2
    rows = [[4, 2], [1, -1], [0, 99], [3, 5]]
    cache = paged.PagedCache(1, 6, 16, kv, d)
    cache.k.fill_(7.0)
    cache.v.fill_(7.0)
    k, v = (torch.full((4, kv, d), x, dtype=BF, device="cuda") for x in (1.0, 2.0))
    paged.append(cache, paged.Step(_i32(rows), _i32([33, 17, 17, 0])), k, v)
    assert (cache.k == 7).all() and (cache.v == 7).all()
    paged.append(cache, paged.Step(_i32(rows), _i32([32, 16, 1, 18])), k, v)
    for b, slot in ((0, 31), (1, 15), (2, 0), (3, 17)):
        p, u = rows[b][slot // 16], slot % 16
        for name, pool, x in (("k", cache.k, 1.0), ("v", cache.v, 2.0)):
            at = ref.slots_of(pool[0], name, [p], 16)
            assert (at[:, u] == x).all()
            at[:, u] = 7.0
            assert (at == 7).all()
    paged.append(cache, paged.Step(_i32(rows), _i32([2, 3, 0, 0]), _i32([0, 4, 4, 4, 4])), k, v)  # a length below its 4 new tokens
    assert (ref.slots_of(cache.k[0], "k", [4], 16)[:, :2] == 1).all() and (ref.slots_of(cache.k[0], "k", [4], 16)[:, 2:] == 7).all()


# ---- attention

@wide_and_narrow
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("d,kv,group", [(64, 2, 1), (96, 1, 8), (128, 2, 8), (128, 1, 3), (192, 2, 5), (256, 1, 17), (64, 1, 40)])
def test_attention_one_token_each(paged, d, kv, group, page):
    f = Filled(paged, [1, 700, 33, 16, 64, 129], kv, d, page, seed=d + group)
    _check(f, paged, _rand(torch.Generator().manual_seed(2), 6, kv * group, d, gain=1.5), None)


@wide_and_narrow
@pytest.mark.parametrize("d,kv,group,counts,lens,page", [
    (64, 2, 4, [40, 0, 1, 200], [40, 9, 500, 333], 16), (128, 1, 8, [130, 33, 1], [130, 900, 64], 32), (96, 3, 2, [65, 64], [65, 1000], 16),
    (192, 1, 6, [50, 3, 70], [51, 3, 400], 64), (256, 2, 5, [40, 90, 1, 0], [700, 90, 1000, 0], 16), (128, 2, 8, [17], [31], 16)])
def test_attention_ragged_chunks(paged, d, kv, group, counts, lens, page):
    f = Filled(paged, lens, kv, d, page, seed=d)
    _check(f, paged, _rand(torch.Generator().manual_seed(3), sum(counts), kv * group, d, gain=1.5), counts)


@wide_and_narrow
@pytest.mark.parametrize("d,kv,group,lens", [(128, 2, 8, [700]), (64, 1, 4, [1300, 20]), (256, 1, 2, [300])])
def test_attention_whole_prompts(paged, d, kv, group, lens):
    f = Filled(paged, lens, kv, d, 16, seed=d)
    _check(f, paged, _rand(torch.Generator().manual_seed(4), sum(lens), kv * group, d, gain=1.5), lens)


def _masks(rng, counts, words, kind):
    rows = []
    for m in counts:
        if kind == "tree":
            parents = [-1] + [rng.randrange(-1, i) for i in range(1, m)]
            rows += ref.plan(parents[:m], m, words)[0]
        elif kind == "any":  # bits of later nodes and past the last one as well
            rows += [[rng.getrandbits(32) for _ in range(words)] for _ in range(m)]
        else:
            rows += [[0] * words for _ in range(m)]
    return rows


@wide_and_narrow
@pytest.mark.parametrize("kind", ["tree", "any", "none"])
@pytest.mark.parametrize("d,kv,group,counts,lens,words", [
    (128, 2, 8, [1, 5, 30], [1, 5, 400], 1), (64, 1, 2, [70, 33, 0], [100, 33, 64], 3), (96, 2, 4, [40, 64], [41, 1000], 2),
    (256, 1, 6, [20, 90], [333, 90], 2), (128, 1, 4, [3, 2], [3, 900], 1), (192, 2, 3, [33, 40], [33, 70], 1)])
def test_attention_under_a_mask(paged, d, kv, group, counts, lens, words, kind):
    """Trees, masks of any bits, and rows that see nothing but what was there before the step (an empty context: nothing)."""
    f = Filled(paged, lens, kv, d, 16, seed=d + words)
    mask = _masks(random.Random(d), counts, words, kind)
    _check(f, paged, _rand(torch.Generator().manual_seed(5), sum(counts), kv * group, d, gain=1.5), counts, mask=mask)


@wide_and_narrow
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d,kv,group,counts,lens,page", [
    (64, 1, 2, [70, 30], [2500, 900], 16), (96, 2, 3, [40, 50], [1700, 3000], 32), (128, 1, 8, [20, 17, 18], [1200, 3100, 5], 16),
    (192, 1, 4, [33], [1500], 64), (256, 2, 2, [60, 9, 70], [640, 1300, 900], 16)])
def test_attention_of_many_rows_over_long_contexts(paged, d, kv, group, counts, lens, page, masked):
    """In a wide table, tiles of 128 rows in several parts; in a narrow one as the sizes have it."""
    counts = [min(m, n) for m, n in zip(counts, lens)]
    f = Filled(paged, lens, kv, d, page, seed=d + 1)
    mask = _masks(random.Random(d), counts, 3, "tree") if masked else None
    _check(f, paged, _rand(torch.Generator().manual_seed(12), sum(counts), kv * group, d, gain=1.5), counts, mask=mask)


@wide_and_narrow
def test_a_chain_under_a_mask_is_the_causal_call(paged):
    counts, lens = [90, 40, 1], [333, 40, 77]
    f = Filled(paged, lens, 2, 128, 16)
    q = _rand(torch.Generator().manual_seed(6), sum(counts), 16, 128)
    step = paged.Step(f.table, f.lengths, _starts(counts))
    parents = _i32([i - 1 for m in counts for i in range(m)])
    mask, positions = paged.tree_plan(parents, f.lengths, step.starts, nodes=90)
    assert positions.tolist() == [n - m + i for m, n in zip(counts, lens) for i in range(m)]
    a, b = paged.attention(f.cache, step, q.cuda()), paged.attention(f.cache, step, q.cuda(), mask=mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@wide_and_narrow
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("m", [1, 60])
def test_lengths_below_the_new_tokens_and_past_the_table(paged, m, masked):
    """Rows whose slot would be before the first see nothing (causal) or what their bits say; slots past the table are not there."""
    d, kv, group = 64, 1, 2
    f = Filled(paged, [96, 96], kv, d, 16, seed=8)  # 7 pages of table, the last one none
    f.lens = [96, 96]
    q = _rand(torch.Generator().manual_seed(7), 2 * m, kv * group, d)
    short, far = max(m - 20, 0), 5000
    f.lengths = _i32([short, far])
    step = paged.Step(f.table, f.lengths, _i32([0, m, 2 * m]))
    mask = torch.full((2 * m, 2), -1, dtype=I32, device="cuda") if masked else None
    out, lse = (x.cpu() for x in paged.attention(f.cache, step, q.cuda(), mask=mask))
    for b, n in ((0, short), (1, far)):
        k, v = f.sequence(b)
        seen = ref.sees(m, n, 96, [[0xFFFFFFFF] * 2] * m if masked else None)
        want, wl, mass, _ = ref.attention(q[b * m: b * m + m], k, v, seen, d ** -0.5)
        assert ((out[b * m: b * m + m].double() - want).abs() <= 2.0 ** -7 * (mass + want.abs())).all()
        assert torch.equal(torch.isneginf(lse[b * m: b * m + m]), torch.isinf(wl))


@wide_and_narrow
@pytest.mark.parametrize("m", [1, 50])
@pytest.mark.parametrize("holes", [[0], [1, 4], [2, 3, 5], [0, 1, 2, 3, 4, 5, 6]])
def test_slots_without_a_page_are_not_seen(paged, m, holes):
    d, kv, group, n = 128, 2, 4, 110
    f = Filled(paged, [n], kv, d, 16, seed=9)
    q = _rand(torch.Generator().manual_seed(8), m, kv * group, d)
    table = f.table.clone()
    for i, p in enumerate(holes):
        table[0, p] = [-1, f.cache.pages, 1 << 30][i % 3]
    out, lse = (x.cpu() for x in paged.attention(f.cache, paged.Step(table, f.lengths, _i32([0, m])), q.cuda()))
    k, v = f.sequence(0)
    seen = ref.sees(m, n, n)
    for p in holes:
        seen[:, 16 * p: 16 * p + 16] = False
    want, wl, mass, _ = ref.attention(q, k, v, seen, d ** -0.5)
    assert ((out.double() - want).abs() <= 2.0 ** -7 * (mass + want.abs())).all()
    assert torch.equal(torch.isneginf(lse), torch.isinf(wl)) and ((lse.double() - wl).abs().nan_to_num(0.0) <= 2.0 ** -18).all()


@wide_and_narrow
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("d,m,masked", [(128, 1, False), (128, 60, False), (64, 3, True), (256, 40, True), (96, 90, False), (192, 2, False)])
def test_infinities_and_nan_stay_with_the_rows_that_see_them(paged, d, m, masked, which, bad):
    kv, group, n = 1, 2, 200
    f = Filled(paged, [n, n], kv, d, 16, seed=10)
    q = _rand(torch.Generator().manual_seed(9), 2 * m, kv * group, d)
    slots = sorted({n - 1, n - 1 - m // 2, n - m})  # of sequence 0: new tokens that some rows see
    for s in slots:
        p, u, x = f.rows[0][s // 16], s % 16, 5 if which == "v" else 3
        pool, at = (f.cache.v, ref.value_at(u, x)) if which == "v" else (f.cache.k, ref.key_at(u, x))
        pool[0, p, 0, 0, at] = bad
    mask = None
    if masked:  # every node sees itself alone
        mask = [[(1 << i) >> (32 * w) & 0xFFFFFFFF for w in range(2)] for i in range(m)] * 2
    gm = None if mask is None else torch.tensor([[x - (1 << 32) if x >> 31 else x for x in r] for r in mask], dtype=I32, device="cuda")
    out, lse = (x.cpu() for x in paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m, 2 * m])), q.cuda(), mask=gm))
    for b in range(2):
        k, v = f.sequence(b)
        seen = ref.sees(m, n, n, None if mask is None else mask[:m])
        want, wl, mass, _ = ref.attention(q[b * m: b * m + m], k, v, seen, d ** -0.5)
        hit = seen[:, slots].any(1) if b == 0 else torch.zeros(m, dtype=torch.bool)
        got, gl = out[b * m: b * m + m], lse[b * m: b * m + m]
        tol = 2.0 ** -7 * (mass + want.abs())
        assert ((got[~hit].double() - want[~hit]).abs() <= tol[~hit]).all() and ((gl[~hit].double() - wl[~hit]).abs() <= 2.0 ** -18).all()
        if which == "v":
            rest = [x for x in range(d) if x != 5]
            assert not torch.isfinite(got[hit][..., 5]).any()
            assert ((got[hit].double() - want[hit]).abs() <= tol[hit])[..., rest].all() and torch.isfinite(gl).all()
            assert math.isnan(bad) or not (got[hit][..., 5] == -bad).any()
        elif math.isnan(bad):
            assert torch.isnan(got[hit]).all() and torch.isnan(gl[hit]).all()
        else:  # a score of +infinity: NaN; of -infinity: a weight of 0
            up = (q[b * m: b * m + m, :, 3].float() * bad > 0)[hit]
            assert torch.isnan(got[hit][up]).all() and not torch.isnan(got[hit][~up]).any()


@wide_and_narrow
@pytest.mark.parametrize("m", [1, 40])
def test_queries_that_are_infinite_or_nan_and_rows_of_no_weight(paged, m):
    d, n = 128, 90
    f = Filled(paged, [n], 1, d, 16, seed=11)
    q = _rand(torch.Generator().manual_seed(10), m, 2, d)
    good = q.clone()
    q[0, 0, 7], q[m - 1, 1, 0] = math.inf, math.nan
    out, lse = (x.cpu() for x in paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m])), q.cuda()))
    plain, pl = (x.cpu() for x in paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m])), good.cuda()))
    hit = torch.zeros(m, 2, dtype=torch.bool)
    hit[0, 0] = hit[m - 1, 1] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], plain[~hit]) and torch.equal(lse[~hit], pl[~hit])
    # scores of -infinity alone: 0 / 0
    k = f.k.clone()
    k[:, 0, 0] = -math.inf
    paged.append(f.cache, paged.Step(f.table, f.lengths, _i32([0, n])), k.cuda(), f.v.cuda())
    q = good.clone()
    q[..., 0] = 1.0
    out, lse = (x.cpu() for x in paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m])), q.cuda()))
    assert torch.isnan(out).all() and torch.isnan(lse).all()


@wide_and_narrow
@pytest.mark.parametrize("scale", [-0.25, 0.0, 1.5])
@pytest.mark.parametrize("m", [1, 50])
def test_attention_at_any_scale(paged, scale, m):
    f = Filled(paged, [300, 70], 2, 64, 32, seed=12)
    _check(f, paged, _rand(torch.Generator().manual_seed(11), 2 * m, 8, 64), [m, m], scale=scale)


@wide_and_narrow
@pytest.mark.parametrize("gain", [1e-30, 1e30])
@pytest.mark.parametrize("m", [1, 50])
def test_attention_range_of_values_and_scores(paged, gain, m):
    """Values of any size; scores of thousands, where the differences between them are what counts."""
    f = Filled(paged, [400], 1, 128, 16, seed=13, gain=gain)
    q = _rand(torch.Generator().manual_seed(12), m, 4, 128)
    _check(f, paged, q, [m])
    _check(f, paged, (q.float() * 200).to(BF), [m])


@wide_and_narrow
def test_equal_scores_of_any_size_average(paged):
    """Keys alike: every weight is 1 / n, whatever the score (2^20 here, from block to block the same)."""
    for m in (1, 40):
        f = Filled(paged, [250], 1, 64, 16, seed=14)
        k = torch.full((250, 1, 64), 128.0, dtype=BF)
        paged.append(f.cache, paged.Step(f.table, f.lengths, _i32([0, 250])), k.cuda(), f.v.cuda())
        f.k = k
        q = torch.full((m, 2, 64), 128.0, dtype=BF)
        out, lse = paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m])), q.cuda(), scale=1.0)
        for i in range(m):
            n = 250 - m + i + 1
            want = f.v[:n, 0].double().mean(0)
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -7 * f.v[:n, 0].double().abs().mean(0)
            assert ((out[i].cpu().double() - want).abs() <= tol).all()
            assert abs(float(lse[i, 0]) - (2.0 ** 20 + math.log(n))) <= 0.25  # two f32 roundings at 2^20


@wide_and_narrow
def test_strided_queries_and_rows_of_nobody(paged, kq):
    """Queries inside the rows of a fused projection; rows before the first and behind the last sequence keep their results."""
    for counts, lens in (([3, 2], [900, 40]), ([90, 30], [200, 300])):
        f = Filled(paged, lens, 2, 128, 16, seed=15)
        t = sum(counts)
        wide = _rand(torch.Generator().manual_seed(13), t + 9, 20, 128).cuda()
        q = wide[:, 3:19]
        starts = _i32([4, 4 + counts[0], 4 + t])
        out, lse = torch.full((t + 9, 16, 128), 7.0, dtype=BF, device="cuda"), torch.full((t + 9, 16), 7.0, device="cuda")
        paged.attention(f.cache, paged.Step(f.table, f.lengths, starts), q, out=out, lse=lse)
        plain, pl = paged.attention(f.cache, paged.Step(f.table, f.lengths, starts), q.contiguous())
        assert torch.equal(out[4: 4 + t], plain[4: 4 + t]) and torch.equal(lse[4: 4 + t], pl[4: 4 + t])
        # the call without the other rows may share its work out otherwise: both are off by their roundings of result and weights
        want, wl = _check(f, paged, q[4: 4 + t].cpu(), counts)
        tol = 2 * 2.0 ** -8 * (1 + 2.0 ** -8) * (want.float().abs() + float(f.v.abs().max()))
        assert ((out[4: 4 + t].cpu().float() - want.float()).abs() <= tol).all() and (lse[4: 4 + t].cpu() - wl).abs().max() <= 2.0 ** -18
        for x in (out, lse):
            assert (x[:4] == 7).all() and (x[4 + t:] == 7).all()
        k = wide[:, :2]
        before = f.cache.k.clone()
        q_out = torch.full((t + 9, 16, 128), 7.0, dtype=BF, device="cuda")
        w = torch.ones(128, dtype=BF, device="cuda")
        paged.append(f.cache, paged.Step(f.table, f.lengths, starts), k, k, q=q[:, :16].contiguous(), q_out=q_out, q_norm=w)
        assert (q_out[:4] == 7).all() and (q_out[4 + t:] == 7).all() and (q_out[4: 4 + t] != 7).any()
        assert not torch.equal(before, f.cache.k)


@wide_and_narrow
@pytest.mark.parametrize("batch", [63, 65, 130, 1100])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_sequences(paged, batch, ragged):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 60, (batch,), generator=g).tolist()
    counts = [min(n, c) for n, c in zip(lens, torch.randint(0, 9, (batch,), generator=g).tolist())] if ragged else None
    f = Filled(paged, lens, 1, 64, 16, seed=16)
    _check(f, paged, _rand(g, sum(counts) if ragged else batch, 4, 64), counts)


@wide_and_narrow
@pytest.mark.parametrize("m", [1, 40])
def test_long_sequences_among_many(paged, m):
    """More sequences than a wave has lanes, two of them long enough to be split."""
    lens = [20 + i % 60 for i in range(90)]
    lens[17], lens[80] = 3000, 2100
    counts = [min(m if i % 9 == 8 else 1, n) for i, n in enumerate(lens)]
    f = Filled(paged, lens, 1, 128, 16, seed=20)
    _check(f, paged, _rand(torch.Generator().manual_seed(21), sum(counts), 4, 128, gain=1.5), counts)


@wide_and_narrow
def test_sequences_share_pages(paged):
    """A prefix that several sequences have in common lies in the pool once."""
    f = Filled(paged, [100, 40, 40], 2, 64, 16, seed=17)
    rows = [r[:] for r in f.rows]
    for b in (1, 2):
        rows[b][:2] = rows[0][:2]
    f.table = _i32(rows)
    for b in (1, 2):
        t0 = sum(f.lens[:b])
        f.k[t0: t0 + 32], f.v[t0: t0 + 32] = f.k[:32], f.v[:32]
    _check(f, paged, _rand(torch.Generator().manual_seed(14), 3, 8, 64), None)
    _check(f, paged, _rand(torch.Generator().manual_seed(15), 75, 8, 64), [40, 20, 15])


def test_pages_beyond_4_gib_and_a_long_context(paged):
    """Pages at the far end of a pool of 6 GB, one sequence of 70000 tokens in them: as in a small pool."""
    n, kv, d, page = 70000, 1, 128, 256
    each = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(18)
    k, v = (torch.randn(n, kv, d, device="cuda", generator=g).to(BF) for _ in "kv")
    q = torch.randn(40, 4, d, device="cuda", generator=g).to(BF)
    got = []
    for pages in (each, 100000):
        cache = paged.PagedCache(1, pages, page, kv, d)
        table = torch.arange(pages - each, pages, dtype=I32, device="cuda").flip(0)[None].contiguous()
        lengths = _i32([n])
        paged.append(cache, paged.Step(table, lengths, _i32([0, n])), k, v)
        for m in (1, 40):
            got.append(paged.attention(cache, paged.Step(table, lengths, _i32([0, m])), q[:m]))
        back = paged.read(cache, paged.Step(table, lengths), 500, first=_i32([n - 500]))
        assert torch.equal(back[0][0], k[-500:]) and torch.equal(back[1][0], v[-500:])
        del cache
    for a, b in zip(got[:2], got[2:]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = (k[:, 0].float() @ q[0].float().t() * d ** -0.5).double()  # [n, heads]
    want = torch.softmax(x, 0).t() @ v[:, 0].double()
    mass = torch.softmax(x, 0).t() @ v[:, 0].double().abs()
    assert ((got[0][0][0].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * mass).all()


@wide_and_narrow
def test_calls_share_a_workspace_and_are_replayed(paged):
    """Eager calls of several shapes and captured ones, in turn over one workspace: every result as alone."""
    shapes = [([1, 1], [900, 40], False), ([30, 9], [400, 77], True), ([200, 1], [300, 3000], False), ([1, 0], [64, 9], False)]
    cases = []
    for i, (counts, lens, masked) in enumerate(shapes):
        f = Filled(paged, lens, 2, 128, 16, seed=20 + i)
        q = _rand(torch.Generator().manual_seed(i), sum(counts), 16, 128).cuda()
        step = paged.Step(f.table, f.lengths, _starts(counts))
        mask = paged.tree_plan(_i32([max(-1, x // 2 - 1) for m in counts for x in range(m)]), f.lengths, step.starts, nodes=max(counts))[0] if masked else None
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        cases.append((f, step, q, mask, out, lse))
    most = max(paged.attention_workspace(f.cache, s, 16, q.shape[0]).numel() for f, s, q, *_ in cases)
    ws = torch.empty(most, dtype=torch.uint8, device="cuda")
    want = [[t.clone() for t in paged.attention(f.cache, s, q, mask=m)] for f, s, q, m, *_ in cases]

    def one(c, space):
        f, s, q, m, out, lse = c
        paged.attention(f.cache, s, q, mask=m, out=out, lse=lse, workspace=space)
    graphs = []
    for c in cases:
        for _ in range(2):
            one(c, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one(c, ws)
        graphs.append(graph)
    for _ in range(4):
        for c, graph, (o, l) in zip(cases, graphs, want):
            c[4].zero_()
            c[5].zero_()
            graph.replay()
            assert torch.equal(c[4], o) and torch.equal(c[5], l)
            ws.random_()
            one(c, ws)
            assert torch.equal(c[4], o) and torch.equal(c[5], l)


@wide_and_narrow
def test_other_streams(paged):
    f = Filled(paged, [3000, 2000], 2, 64, 16, seed=30)
    q, starts = _rand(torch.Generator().manual_seed(30), 400, 8, 64).cuda(), _starts([300, 100])
    step = paged.Step(f.table, f.lengths, starts)
    want = paged.attention(f.cache, step, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        got = paged.attention(f.cache, step, q, stream=stream)
        back = paged.read(f.cache, step, 50, stream=stream)
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(back[0][0], f.k[:50].cuda())
    with torch.cuda.stream(side):
        got = paged.attention(f.cache, step, q)
    side.synchronize()
    assert torch.equal(got[0], want[0])


def test_binding_refuses(paged, kq):
    f = Filled(paged, [20, 9], 2, 64, 16, seed=31)
    step, q = paged.Step(f.table, f.lengths), torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    bad = [lambda: paged.attention(f.cache, step, q.float()), lambda: paged.attention(f.cache, step, q[..., :32]),
           lambda: paged.attention(f.cache, step, q, mask=torch.zeros(3, 1, dtype=I32, device="cuda")),
           lambda: paged.attention(f.cache, step, q, mask=torch.zeros(2, 1, device="cuda")),
           lambda: paged.attention(f.cache, step, q, mask=torch.zeros(2, 0, dtype=I32, device="cuda")),
           lambda: paged.attention(f.cache, step, q, out=q[:1]), lambda: paged.attention(f.cache, step, q.transpose(0, 1)),
           lambda: paged.append(f.cache, step, k, k[:1]), lambda: paged.append(f.cache, step, k[:, :1], k[:, :1]),
           lambda: paged.append(f.cache, step, k, k, cos_sin=torch.zeros(4, 32, 2, device="cuda")),
           lambda: paged.append(f.cache, step, k, k, q=q[:1], q_norm=torch.ones(64, dtype=BF, device="cuda")),
           lambda: paged.append(f.cache, step, k, k, k_norm=torch.ones(64, device="cuda")),
           lambda: paged.read(f.cache, step, 4, dtype=torch.float16), lambda: paged.Step(f.table, f.lengths, _i32([0, 1])),
           lambda: paged.Step(f.table.float(), f.lengths), lambda: paged.Step(f.table, f.lengths[:1]),
           lambda: paged.tree_plan(_i32([-1, 0]), f.lengths), lambda: paged.tree_plan(_i32([-1, 0]), f.lengths, nodes=0),
           lambda: paged.commit(f.cache, step, _i32([1, 2]), _i32([-1]), _i32([1, 2])),
           lambda: paged.commit(f.cache, step, _i32([1, 2]), _i32([-1, -1]), _i32([1, 2]), counts=_i32([0]))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: paged.attention(f.cache, step, q, layer=1), lambda: paged.attention(f.cache, step, q[:1]),
                 lambda: paged.append(f.cache, step, k, k, q=q), lambda: paged.attention(f.cache, step, q[:, :3].contiguous()),
                 lambda: paged.commit(f.cache, step, _i32([1, 2]), _i32([-1, -1]), _i32([1, 2]), new_lengths=f.lengths)):
        with pytest.raises(kq.KrError):
            call()
