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
