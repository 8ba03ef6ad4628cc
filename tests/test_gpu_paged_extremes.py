"""GPU: infinities and NaN among the values of slots that every row sees, over the paged cache: what the formula gives."""
import math

import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import Filled, _check, _i32, _rand, paged, table_of, wide_and_narrow  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@wide_and_narrow
@pytest.mark.parametrize("d,m,n", [(64, 1, 200), (96, 3, 100), (128, 1, 3000), (192, 2, 200), (256, 1, 700), (128, 60, 400), (64, 90, 3000), (256, 40, 1300)])
def test_infinite_values_that_every_row_sees(paged, d, m, n):
    """One infinity of a dim: that infinity in every row; two alike: the same; both, or a NaN: NaN.  The other dims and lse are
    as they would be without them (under the bound of test_gpu_paged's _check, whose values they replace)."""
    kv, group = 1, 2
    f = Filled(paged, [n, n], kv, d, 16, seed=d + m)
    q = _rand(torch.Generator().manual_seed(m), 2 * m, kv * group, d)
    clean, clean_lse = _check(f, paged, q, [m, m])
    bad = {3: [(5, INF)], 7: [(20, -INF)], 11: [(1, INF), (n - m - 1, INF)], 30: [(40, -INF), (41, -INF)], 40: [(9, INF), (33, -INF)], 41: [(17, NAN)],
           42: [(2, NAN), (60, INF)]}
    for x, at in bad.items():
        for slot, value in at:
            assert slot < n - m  # every row of the sequence sees it
            f.cache.v[0, f.rows[0][slot // 16], 0, 0, ref.value_at(slot % 16, x)] = value
    out, lse = (t.cpu() for t in paged.attention(f.cache, paged.Step(f.table, f.lengths, _i32([0, m, 2 * m])), q.cuda()))
    for x, at in bad.items():
        got, want = out[:m, :, x], sum(v for _, v in at)
        assert torch.isnan(got).all() if math.isnan(want) else (got == want).all(), (x, at, got.flatten()[:8])
    rest = [x for x in range(d) if x not in bad]
    assert torch.equal(out[:m][..., rest], clean[:m][..., rest]) and torch.equal(lse, clean_lse) and torch.equal(out[m:], clean[m:])
