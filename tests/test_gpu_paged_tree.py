"""GPU: plans of trees of drafted tokens and commits of their accepted paths against their definitions."""
import random

import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import Filled, _i32, _starts, paged  # noqa: F401  (paged: the fixture)

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _unsigned(mask):
    return [[x & 0xFFFFFFFF for x in row] for row in mask.tolist()]


def _tree(rng, m, kind):
    if kind == "chain":
        return [i - 1 for i in range(m)]
    if kind == "star":
        return [-1] + [0] * (m - 1)
    if kind == "wild":  # parents that are none: itself, later nodes, far ones
        return [rng.choice([-1, -7, i, i + 1, 1 << 30, rng.randrange(i + 1), rng.randrange(i + 1)]) for i in range(m)]
    return [-1] + [i - 1 if rng.random() < 0.5 else rng.randrange(-1, i) for i in range(1, m)]


@pytest.mark.parametrize("kind", ["tree", "chain", "star", "wild"])
@pytest.mark.parametrize("counts,words", [([1], 1), ([24, 0, 33], 2), ([64, 65, 1, 300], 10), ([100, 20], 1), ([2000, 7], 63), ([4100], 128)])
def test_plan(paged, counts, words, kind):
    rng = random.Random(len(counts) + words)
    trees = [_tree(rng, m, kind)[:m] for m in counts]
    lens = [m + rng.randrange(0, 500) for m in counts]
    t = sum(counts)
    mask, positions = (torch.full(s, 77, dtype=I32, device="cuda") for s in ((t + 2, words), (t + 2,)))
    starts = _starts(counts)
    paged.tree_plan(_i32([p for x in trees for p in x] + [5, 5]), _i32(lens), starts, mask=mask, positions=positions)
    t0 = 0
    got, at = _unsigned(mask), positions.tolist()
    for x, n in zip(trees, lens):
        rows, where = ref.plan(x, n, words)
        assert got[t0: t0 + len(x)] == rows and at[t0: t0 + len(x)] == where
        t0 += len(x)
    assert (mask[t:] == 77).all() and (positions[t:] == 77).all()  # nobody's rows


def test_plan_without_starts(paged):
    mask, positions = paged.tree_plan(_i32([-1, -1, 0]), _i32([5, 1, 9]), nodes=40)
    assert _unsigned(mask) == [[1, 0]] * 3 and positions.tolist() == [4, 0, 8]


def _choices(rng, parents, stop):
    tokens = [rng.randrange(50) for _ in parents]
    targets = [rng.randrange(50) for _ in parents]
    at = 0
    while rng.random() > stop:
        children = [i for i, p in enumerate(parents) if p == at and i > at]
        if not children:
            break
        child = rng.choice(children)
        targets[at] = tokens[child]
        at = next(i for i in children if tokens[i] == tokens[child])
    return tokens, targets


@pytest.mark.parametrize("d,kv,page,layers", [(64, 1, 16, 1), (128, 2, 16, 5), (96, 3, 32, 2), (192, 1, 64, 3), (256, 2, 16, 2)])
@pytest.mark.parametrize("counts,most,kind", [([1], 4, "tree"), ([24, 0, 40, 3], 32, "tree"), ([90, 200], 7, "tree"), ([70, 30], 64, "chain"),
                                               ([40, 9], 16, "wild"), ([33], 1, "tree")])
def test_commit(paged, d, kv, page, layers, counts, most, kind):
    """Paths, counts, the next tokens, and every slot of every layer."""
    rng = random.Random(d + most)
    lens = [m + rng.randrange(0, 90) for m in counts]
    f = Filled(paged, lens, kv, d, page, seed=d, layers=layers)
    trees = [_tree(rng, m, kind)[:m] for m in counts]
    choices = [_choices(rng, x, 0.02) for x in trees]
    flat = lambda xs: _i32([v for x in xs for v in x])  # noqa: E731
    before = f.cache.k.clone(), f.cache.v.clone()
    nxt = torch.full((len(counts),), 99, dtype=I32, device="cuda")
    path, kept, nxt, new = paged.commit(f.cache, paged.Step(f.table, f.lengths, _starts(counts)), flat(c[0] for c in choices), flat(trees),
                                        flat(c[1] for c in choices), next=nxt, max_path=most)
    for b, (m, n) in enumerate(zip(counts, lens)):
        want = ref.path(choices[b][0], [p if 0 <= p < i else -1 for i, p in enumerate(trees[b])], choices[b][1], most)
        assert path[b].tolist() == want + [0] * (most - len(want)) and int(kept[b]) == len(want) and int(new[b]) == n - m + len(want)
        assert int(nxt[b]) == (choices[b][1][want[-1]] if m else 99)
        for layer in range(layers):
            for name, pool, old in (("k", f.cache.k, before[0]), ("v", f.cache.v, before[1])):
                was, now = (ref.slots_of(x[layer], name, f.pages(b), page) for x in (old, pool))
                for i, node in enumerate(want):
                    was[:, n - m + i] = ref.slots_of(old[layer], name, f.pages(b), page)[:, n - m + node]
                assert torch.equal(was.nan_to_num(1e9), now.nan_to_num(1e9))
    # pages of nobody
    used = {p for r in f.rows for p in r}
    for p in set(range(f.cache.pages)) - used:
        assert torch.equal(f.cache.k[:, p].view(torch.int16), before[0][:, p].view(torch.int16))


def test_commit_cut_off_and_missing_pages(paged):
    """A length below its new tokens, slots past the table and without a page: no move, the path is found all the same."""
    f = Filled(paged, [32, 32], 1, 64, 16, seed=3)
    rows = [f.rows[0][:2], [-1, f.rows[1][1]]]
    before = f.cache.k.clone(), f.cache.v.clone()
    parents, tokens, targets = [-1, 0, 0, 2] * 2, [1, 2, 3, 4] * 2, [3, 9, 4, 8] * 2
    step = paged.Step(_i32(rows), _i32([2, 18]), _i32([0, 4, 8]))
    path, counts, nxt, new = paged.commit(f.cache, step, _i32(tokens), _i32(parents), _i32(targets), max_path=5)
    assert path.tolist() == [[0, 2, 3, 0, 0]] * 2 and counts.tolist() == [3, 3] and nxt.tolist() == [8, 8] and new.tolist() == [1, 17]
    for a, b in zip(before, (f.cache.k, f.cache.v)):  # sequence 1: slots 14 .. 17, of which the first two have no page
        assert torch.equal(a[:, f.rows[0][:2]].view(torch.int16), b[:, f.rows[0][:2]].view(torch.int16))
        assert torch.equal(a[:, f.rows[1][0]].view(torch.int16), b[:, f.rows[1][0]].view(torch.int16))
    was, now = (ref.slots_of(x[0], "v", [f.rows[1][1]], 16) for x in (before[1], f.cache.v))
    was[:, 0] = was[:, 1]  # node 3 (slot 17) to slot 16
    assert torch.equal(was.nan_to_num(1e9), now.nan_to_num(1e9))


def test_a_drafted_step_is_the_same_as_its_tokens_one_by_one(paged):
    """Append a tree, attend under its plan, commit: the accepted rows' results and the cache are those of plain decoding, bit for bit
    where the launches are alike; captured and replayed over new trees too."""
    from kriya_q4 import rope

    d, kv, heads, page, layers, batch, m = 64, 2, 8, 16, 2, 2, 12
    g = torch.Generator().manual_seed(5)
    lens = [50, 33]
    f = Filled(paged, lens, kv, d, page, seed=5, layers=layers, spare=8)
    free = [p for p in range(f.cache.pages) if all(p not in r for r in f.rows)]
    table = _i32([[p for p in r if p >= 0] + free[4 * b: 4 * b + 4] + [-1] * (5 - -(-n // page)) for b, (r, n) in enumerate(zip(f.rows, lens))])
    for layer in range(layers):
        paged.append(f.cache, paged.Step(table, f.lengths, _starts(lens)), f.k.cuda(), f.v.cuda(), layer)
    cs = rope.table(d, 200, 1e4)
    lengths, starts = _i32([n + m for n in lens]), _i32([0, m, 2 * m])
    parents, tokens, targets = (torch.zeros(2 * m, dtype=I32, device="cuda") for _ in range(3))
    k, v, q = ((torch.randn(2 * m, x, d, generator=g)).to(torch.bfloat16).cuda() for x in (kv, kv, heads))
    q_out, mask, positions = torch.empty_like(q), torch.empty(2 * m, 1, dtype=I32, device="cuda"), torch.empty(2 * m, dtype=I32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(2 * m, heads, device="cuda")
    path, counts, nxt, new = (torch.zeros(s, dtype=I32, device="cuda") for s in ((2, 8), (2,), (2,), (2,)))
    step = paged.Step(table, lengths, starts)
    ws = paged.attention_workspace(f.cache, step, heads, 2 * m)

    def run():
        paged.tree_plan(parents, lengths, starts, mask=mask, positions=positions)
        for layer in range(layers):
            paged.append(f.cache, step, k, v, layer, q=q, q_out=q_out, cos_sin=cs, positions=positions)
            paged.attention(f.cache, step, q_out, layer, mask=mask, out=out, lse=lse, workspace=ws)
        paged.commit(f.cache, step, tokens, parents, targets, path, counts, nxt, new)
    pool = f.cache.k.clone(), f.cache.v.clone()
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(3):
        rng = random.Random(seed)
        trees = [_tree(rng, m, "tree") for _ in lens]
        for x in trees:
            x[0] = -1
        choices = [_choices(rng, x, 0.05) for x in trees]
        for to, xs in ((parents, trees), (tokens, [c[0] for c in choices]), (targets, [c[1] for c in choices])):
            to.copy_(_i32([y for x in xs for y in x]))
        for captured in (False, True):
            f.cache.k.copy_(pool[0])
            f.cache.v.copy_(pool[1])
            graph.replay() if captured else run()
            torch.cuda.synchronize()
            for b in range(batch):
                want = ref.path(choices[b][0], trees[b], choices[b][1], 8)
                n = int(counts[b])
                assert path[b, :n].tolist() == want and int(new[b]) == lens[b] + n
                # the same tokens one after the other, into a copy
                other = paged.PagedCache.wrap(pool[0].clone(), pool[1].clone())
                for i, node in enumerate(want):
                    at = _i32([lens[b] + i + 1])
                    one = paged.Step(table[b: b + 1], at)
                    row = b * m + node
                    qq = torch.empty_like(q[:1])
                    for layer in range(layers):
                        paged.append(other, one, k[row: row + 1], v[row: row + 1], layer, q=q[row: row + 1], q_out=qq, cos_sin=cs, positions=at - 1)
                        o, s = paged.attention(other, one, qq, layer)
                    assert torch.equal(qq[0], q_out[row])
                    # each off by the rounding of its result and of its weights, whose mean of |v| is at most the largest
                    tol = 2 * 2.0 ** -8 * (1 + 2.0 ** -8) * (o[0].float().abs() + max(float(f.v.abs().max()), float(v.abs().max())))
                    assert ((o[0].float() - out[row].float()).abs() <= tol).all() and (s[0] - lse[row]).abs().max() <= 2.0 ** -18
                a = paged.read(f.cache, paged.Step(table, new), 80, 1)
                c = paged.read(other, paged.Step(table, new), 80, 1)
                assert torch.equal(a[0][b], c[0][b]) and torch.equal(a[1][b], c[1][b])
