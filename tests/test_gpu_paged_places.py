"""GPU: arguments of the paged cache's calls that begin inside a tensor."""
import pytest
import torch

from test_gpu_paged import BF, _i32, _rand, _starts, _table, paged  # noqa: F401  (paged: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary,layout", [(0, 0), (64, 0), (64, 1), (36, 0)])
@pytest.mark.parametrize("at", [1, 2, 4, 7])
def test_norm_weights_at_any_element(paged, at, rotary, layout):
    """The weights of heads need no more alignment than their elements: the same bits as from a tensor of their own."""
    from kriya_q4 import rope

    d, kv, heads, lens = 64, 2, 6, [40, 3]
    g = torch.Generator().manual_seed(at)
    rows, pages = _table(lens, 16, 1)
    step = paged.Step(_i32(rows), _i32(lens), _starts(lens))
    k, v, q = (_rand(g, 43, h, d).cuda() for h in (kv, kv, heads))
    wide = torch.full((2, d + 16), 9.0, dtype=BF, device="cuda")
    wide[:, at: at + d] = (1 + 0.1 * torch.randn(2, d, generator=g)).to(BF).cuda()
    cs, pos = (rope.table(rotary, 60, 1e4), torch.arange(43, dtype=torch.int32, device="cuda")) if rotary else (None, None)
    got = []
    for weights in (wide[:, at: at + d], [w.clone() for w in wide[:, at: at + d]]):
        cache = paged.PagedCache(1, pages, 16, kv, d)
        cache.k.zero_(), cache.v.zero_()
        q_out = torch.empty_like(q)
        paged.append(cache, step, k, v, q=q, q_out=q_out, cos_sin=cs, positions=pos, layout=layout, q_norm=weights[0], k_norm=weights[1])
        got.append((cache.k, q_out))
    assert wide[0, at:].data_ptr() % 16 == 2 * at
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("extra", [0, 3])
def test_rows_in_one_anothers_gaps(paged, extra):
    """k, v, q and q_out in the rows of one tensor, and of one with rows of another length over the same memory: as from tensors apart."""
    d, kv, heads, lens = 64, 2, 4, [30, 5]
    g = torch.Generator().manual_seed(extra)
    rows, pages = _table(lens, 16, 1)
    step = paged.Step(_i32(rows), _i32(lens), _starts(lens))
    wide = _rand(g, 35, 2 * kv + 2 * heads + extra, d).cuda()
    k, v, q, q_out = wide[:, :kv], wide[:, kv: 2 * kv], wide[:, 2 * kv: 2 * kv + heads], wide[:, 2 * kv + heads: 2 * kv + 2 * heads]
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(BF).cuda()
    caches = [paged.PagedCache(1, pages, 16, kv, d) for _ in range(2)]
    for c in caches:
        c.k.zero_(), c.v.zero_()
    apart = [x.contiguous() for x in (k, v, q)]
    paged.append(caches[0], step, *apart[:2], q=apart[2], q_norm=w, k_norm=w)
    paged.append(caches[1], step, k, v, q=q, q_out=q_out, q_norm=w, k_norm=w)
    assert torch.equal(q_out, apart[2]) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    paged.append(caches[1], step, k, v, q=q, q_norm=w, k_norm=w)  # in place
    assert torch.equal(q, apart[2]) and torch.equal(caches[0].k, caches[1].k)


def test_rows_of_other_lengths_in_the_gaps(paged):
    """k and v in rows of 256 elements, q and q_out in rows of 512 where those leave room."""
    d = 64
    block = _rand(torch.Generator().manual_seed(4), 2048).cuda()
    k, v = (block.as_strided((4, 1, d), (256, d, 1), x) for x in (0, 64))
    q, q_out = (block.as_strided((4, 1, d), (512, d, 1), x) for x in (128, 192))
    before, want, w = block.clone(), q.clone(), torch.ones(d, dtype=BF, device="cuda")
    cache = paged.PagedCache(1, 4, 16, 1, d)
    step = paged.Step(_i32([[2, 1]]), _i32([4]), _i32([0, 4]))
    paged.append(cache, step, k, v, q=q, q_out=q_out, q_norm=w)
    paged.append(cache, step, k, v, q=want, q_norm=w)
    assert torch.equal(q_out, want)
    before.as_strided((4, 1, d), (512, d, 1), 192).copy_(want)
    assert torch.equal(block, before)
