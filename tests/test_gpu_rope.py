"""GPU: rotary tables and the rotation in general form against 64 bits."""
import math

import pytest
import torch

import _kv8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rope(kq):
    from kriya_q4 import rope

    return rope


def _freq(r, theta, kind, factor, ctx, slow, fast):
    f = []
    for i in range(r // 2):
        t = theta * factor ** (r / (r - 2)) if kind == "ntk" else theta
        w = t ** (-2 * i / r)
        if kind == "linear":
            w /= factor
        if kind == "parts":
            g = min(max((ctx * w / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0)
            w = w * g + w / factor * (1 - g)
        f.append(w)
    return torch.tensor(f, dtype=torch.float64)


@pytest.mark.parametrize("kind", ["none", "linear", "ntk", "parts"])
@pytest.mark.parametrize("r,first,count,theta", [(128, 0, 70, 1e6), (2, 5, 3, 1e4), (6, 0, 1, 1e4), (64, 1 << 20, 33, 1e4),
                                                 (256, (1 << 32) - 9, 9, 5e5)])
def test_table(rope, kind, r, first, count, theta):
    if kind == "ntk" and r == 2:
        r = 4  # a single pair has no such scaling
    z = rope.Scaling(kind, 8.0, 4096, 1.0, 32.0, 1.25)
    got = rope.table(r, count, theta, first=first, scaling=z).cpu().double()
    pos = torch.arange(first, first + count, dtype=torch.float64)
    a = pos[:, None] * _freq(r, theta, kind, 8.0, 4096, 1.0, 32.0)
    want = 1.25 * torch.stack([torch.cos(a), torch.sin(a)], -1)
    # the fraction of a turn in f32 (2^-25 of at most half a turn), sine and cosine to 2 ulp; the angle in 64 bits: both
    # sides round frequency and product, 4 roundings of 2^-53 of up to p radians
    tol = 1.25 * (2 * math.pi * 2.0 ** -26 + 2.0 ** -22) + 1.25 * 8 * 2.0 ** -53 * float(pos[-1] + 1)
    assert (got - want).abs().max() <= tol


CASES = [  # tokens, heads, head_dim, rotary, layout, extra elements between tokens
    (1, 1, 64, 64, 0, 0), (5, 3, 128, 128, 0, 256), (3, 18, 128, 128, 1, 0), (7, 2, 128, 32, 0, 128), (4, 5, 96, 48, 1, 8),
    (2, 3, 80, 20, 0, 0), (3, 2, 64, 36, 1, 3), (2, 1, 6, 2, 0, 1), (1, 40, 256, 64, 0, 0), (130, 1, 64, 16, 0, 0)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_apply_in_place_and_out(rope, case, dt):
    t, h, d, r, layout, extra = case
    g = torch.Generator().manual_seed(sum(case))
    buf = torch.randn(t, h * d + extra, generator=g).to(dt)
    x = buf[:, : h * d].unflatten(1, (h, d))
    rows = 50
    table = torch.randn(rows, r // 2, 2, generator=g)
    pos = torch.randint(0, rows, (t,), generator=g, dtype=torch.int32)
    pos[0] = rows - 1
    if t > 2:
        pos[1], pos[2] = rows, -1  # past the table (as u32): not rotated
    cs, pd = table.cuda(), pos.cuda()
    for inverse in (False, True):
        want = ref.rope64(x, table, pos, layout, inverse)
        # f32: two products and a sum, each 2^-24 of its size; then one rounding to the type
        size = ref.rope64(x.double().abs(), table.abs(), pos, layout, True).abs() + want.abs()
        tol = 2.0 ** -22 * (size + x.double().abs() * 4) + (2.0 ** -8 if dt == torch.bfloat16 else 0) * want.abs()
        dev = buf.cuda()
        src = dev[:, : h * d].unflatten(1, (h, d))
        out = torch.full((t, h, d), 7.0, dtype=dt, device="cuda")
        assert rope.apply(src, cs, pd, layout=layout, inverse=inverse, out=out) is out
        assert (torch.equal(dev.cpu(), buf))  # the input stays
        assert ((out.cpu().double() - want).abs() <= tol).all()
        rope.apply(src, cs, pd, layout=layout, inverse=inverse)
        assert torch.equal(src.cpu(), out.cpu())  # in place: the same bits
        assert torch.equal(dev[:, h * d:].cpu(), buf[:, h * d:])  # what lies between the tokens stays
        assert torch.equal(out[..., r:].cpu(), x[..., r:])


def test_inverse_is_the_gradient(rope):
    """d/dx of sum(w . rope(x)) is rope^-1(w): against differences of the 64-bit rotation (linear, so exact)."""
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(3, 2, 64, generator=g), torch.randn(3, 2, 64, generator=g)
    table = torch.randn(9, 16, 2, generator=g)
    pos = torch.tensor([0, 8, 3], dtype=torch.int32)
    got = rope.apply(w.cuda(), table.cuda(), pos.cuda(), inverse=True, out=torch.empty(3, 2, 64, device="cuda")).cpu()
    for i in (0, 5, 15, 16, 31, 32, 63):
        e = torch.zeros_like(x)
        e[1, 1, i] = 1.0
        diff = (w.double() * (ref.rope64(x.double() + e, table, pos, 0) - ref.rope64(x, table, pos, 0))).sum()
        assert abs(float(got[1, 1, i]) - float(diff)) <= 2.0 ** -20 * 8


def test_many_tokens_and_another_stream(rope):
    t, h, d = 3907, 2, 64
    x = torch.randn(t, h, d).to(torch.bfloat16)
    table = rope.table(64, t, 1e4)
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xd = x.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = rope.apply(xd, table, pos, out=torch.empty_like(xd))
    side.synchronize()
    want = ref.rope64(x[-3:], table.cpu(), pos[-3:].cpu(), 0)
    assert ((y[-3:].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all()


def test_binding_refuses(rope):
    x, cs, pos = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(4, 32, 2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        rope.apply(x.to(torch.float16), cs, pos)
    with pytest.raises(ValueError):
        rope.apply(x.transpose(1, 2), cs, pos)
    with pytest.raises(ValueError):
        rope.apply(x, cs, pos[:1])
    with pytest.raises(ValueError):
        rope.apply(x, cs.transpose(0, 1), pos)
    with pytest.raises(ValueError):
        rope.apply(x, cs, pos.long())
    with pytest.raises(RuntimeError, match="rotary_dim"):
        rope.apply(x, torch.zeros(4, 33, 2, device="cuda"), pos)
    with pytest.raises(RuntimeError, match="overlap"):
        rope.apply(torch.zeros(128, device="cuda").as_strided((2, 1, 64), (32, 64, 1)), cs, pos)
    with pytest.raises(RuntimeError, match="different strides"):  # the same memory with tokens elsewhere
        buf = torch.zeros(256, device="cuda")
        rope.apply(buf.view(4, 1, 64)[:2], cs, pos, out=buf.view(2, 1, 128)[..., :64])
