"""The weights of attention over the paged cache where rows are few: two bf16 each, off by at most 2^-16 of themselves (half a step of
bf16, 2^-8, of what half a step leaves).  On the GPU under that bound; on the CPU, that the same cases' results with weights in one
bf16 would not keep it."""
import math

import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import BF, Filled, _check, _rand, paged, table_of, wide_and_narrow  # noqa: F401  (fixtures)

P_HALF = 2.0 ** -16
# head_dim, kv heads, group, new tokens (None: one each), lengths; queries of this gain: scores near 0, so that their own errors are small
CASES = [(64, 2, 4, None, [60, 33, 64]), (96, 1, 8, None, [50, 64]), (128, 2, 8, None, [64, 40]), (192, 1, 3, None, [60]), (256, 1, 16, None, [48, 64]),
         (128, 1, 4, [4, 3], [60, 64]), (64, 2, 2, [8], [64])]
GAIN = 0.2


def _queries(case):
    d, kv, group, counts, lens = case
    return _rand(torch.Generator().manual_seed(d), sum(counts) if counts else len(lens), kv * group, d, gain=GAIN)


@pytest.mark.gpu
@wide_and_narrow
@pytest.mark.parametrize("case", CASES)
def test_weights_keep_two_bf16(paged, case):
    d, kv, group, counts, lens = case
    _check(Filled(paged, lens, kv, d, 16, seed=d + group), paged, _queries(case), counts, p_half=P_HALF)


@pytest.mark.parametrize("case", CASES)
def test_one_bf16_would_be_seen(case):
    """The same inputs with weights rounded to one bf16, in 64 bits otherwise: outside the bound somewhere; to two: inside, with
    all of f32's part of the bound to spare."""
    d, kv, group, counts, lens = case
    g = torch.Generator().manual_seed(d + group)
    q = _queries(case)
    worst = {1: -math.inf, 2: -math.inf}
    for b, (t0, m, n) in enumerate(ref.spans(None if counts is None else [sum(counts[:i]) for i in range(len(counts) + 1)], lens)):
        k, v = (_rand(g, n, kv, d).transpose(0, 1).double() for _ in "kv")
        want, _, mass, terms = ref.attention(q[t0: t0 + m], k, v, ref.sees(m, n, n), d ** -0.5)
        off = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -22
        p = P_HALF + 2 * off[..., None] + 4 * n * 2.0 ** -24
        tol = 2.0 ** -8 * (1 + p) * want.abs() + (1 + 2.0 ** -8) * p * mass
        for pieces in worst:
            for i in range(m):
                for h in range(kv * group):
                    x = (k[h // group, : n - m + i + 1] @ q[t0 + i, h].double()) * d ** -0.5
                    e = torch.exp(x - x.max())
                    used, left = torch.zeros_like(e), e
                    for _ in range(pieces):
                        used, left = used + left.to(BF).double(), left - left.to(BF).double()
                    got = ((used / e.sum()) @ v[h // group, : n - m + i + 1]).to(BF).double()
                    bound = tol[i, h] if pieces == 1 else 2.0 ** -8 * want[i, h].abs() * (1 + P_HALF) + (1 + 2.0 ** -8) * P_HALF * mass[i, h]
                    worst[pieces] = max(worst[pieces], float(((got - want[i, h]).abs() - bound).max()))
    assert worst[1] > 0 >= worst[2], worst
