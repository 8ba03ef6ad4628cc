"""GPU: rotary tables hold the f32 values nearest to the 64-bit ones."""
import math

import pytest
import torch

from test_gpu_rope import _freq, rope  # noqa: F401  (rope: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,gain", [("none", 1.0), ("ntk", 1.25), ("parts", 0.1 * math.log(8.0) + 1.0)])
@pytest.mark.parametrize("r,first,count,theta", [(128, 0, 4000, 1e6), (32, 1 << 20, 333, 1e4)])
def test_table_is_rounded_once(rope, kind, gain, r, first, count, theta):
    got = rope.table(r, count, theta, first=first, scaling=rope.Scaling(kind, 8.0, 4096, 1.0, 32.0, gain)).cpu().double()
    pos = torch.arange(first, first + count, dtype=torch.float64)
    a = pos[:, None] * _freq(r, theta, kind, 8.0, 4096, 1.0, 32.0)
    want = gain * torch.stack([torch.cos(a), torch.sin(a)], -1)
    # half a step of f32; the angle in 64 bits: both sides round frequency and product, 4 roundings of 2^-53 of up to p radians
    tol = 2.0 ** -24 * want.abs() + 2 * 8 * 2.0 ** -53 * float(pos[-1] + 1)
    assert ((got - want).abs() <= tol).all()
