"""GPU: what kr_kv8_append does with query rows that belong to no sequence."""
import pytest
import torch

from test_gpu_kv8 import _i32, _rand, _starts, kv8  # noqa: F401  (kv8: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,counts,lens", [(0, [1, 1], [9, 40]), (0, [40, 0], [40, 9]), (3, [2, 60], [2, 70])])
@pytest.mark.parametrize("rotary", [64, 36])
def test_append_leaves_queries_of_no_sequence_as_they_were(kv8, first, counts, lens, rotary):
    """Rows before the first sequence's and behind the last's are nobody's: q_out, or q in place, keeps what it held there."""
    from kriya_q4 import rope

    g = torch.Generator().manual_seed(first + sum(counts))
    n = first + sum(counts)
    k, v, q = _rand(g, n + 7, 2, 64).cuda(), _rand(g, n + 7, 2, 64).cuda(), _rand(g, n + 7, 4, 64).cuda()
    table, pos = rope.table(rotary, 200, 1e4), torch.randint(1, 200, (n + 7,), generator=g, dtype=torch.int32).cuda()
    want = rope.apply(q, table, pos, out=torch.empty_like(q))
    starts, cache = _starts(counts) + first, kv8.Kv8Cache(2, 2, 64, 80)
    for out in (torch.full_like(q, 3.0), q.clone()):
        before, src = out.clone(), q if (out == 3.0).all() else out
        kv8.append(cache, k, v, _i32(lens), starts=starts, q=src, q_out=out, cos_sin=table, positions=pos)
        assert torch.equal(out[first:n], want[first:n])
        assert torch.equal(out[:first], before[:first]) and torch.equal(out[n:], before[n:])
