"""GPU: attention over the paged cache where the sizes of a launch say little about what its sequences hold, against 64 bits."""
import pytest
import torch

from test_gpu_paged import Filled, _check, _rand, paged  # noqa: F401  (paged: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,counts,lens", [(2000, [1000, 1000], [1500, 1100]), (2000, [1, 0, 1999], [3000, 0, 2100]), (1600, [1600], [2000])])
def test_a_large_batch_of_which_few_sequences_have_tokens(paged, batch, counts, lens):
    """The launch has a workgroup for the tiles that so many sequences could have, and splits the few tiles there are into as many
    parts as have a place in the workspace."""
    counts, lens = ([0] * (batch - len(x) - 1) + x + [0] for x in (counts, lens))
    f = Filled(paged, lens, 1, 64, 16, seed=batch)
    _check(f, paged, _rand(torch.Generator().manual_seed(1), sum(counts), 4, 64, gain=1.5), counts)
