"""GPU: what the 8-bit cache's calls must leave alone: query rows that belong to no sequence, and workspaces of launches whose
tiles stay whole."""
import pytest
import torch

from test_gpu_kv8 import _check_attention, _fill, _i32, _rand, _starts, kv8  # noqa: F401  (kv8: the fixture)

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


@pytest.mark.parametrize("d,kv,group,counts,lens", [
    (64, 2, 4, [200], [200]), (128, 2, 8, [500], [500]), (256, 1, 4, [150, 0, 40], [150, 5, 300]), (64, 1, 40, [3], [9])])
def test_tiles_that_stay_whole_take_nothing_from_the_workspace(kv8, d, kv, group, counts, lens):
    """Launches that may split their tiles and find the contexts too short for it: the same bits whatever the workspace holds."""
    g = torch.Generator().manual_seed(d + sum(counts))
    cache = _fill(kv8, g, lens, kv, d, 0, 6000)
    q, starts, lengths = _rand(g, sum(counts), kv * group, d), _starts(counts), _i32(lens)
    ws, got = kv8.attention_workspace(cache, kv * group, sum(counts)), []
    assert ws.numel() > 16  # (a launch that has parts)
    for byte in (0x00, 0x41, 0xFF):  # zeros, floats near 12, NaN
        got.append(_check_attention(kv8, cache, q, starts, lengths, workspace=ws.fill_(byte))[:2])
    assert all(torch.equal(x, y) for other in got[1:] for x, y in zip(got[0], other))
