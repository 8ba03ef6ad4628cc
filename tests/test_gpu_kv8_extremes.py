"""GPU: attention over the 8-bit cache and its weights at the ends of the range, against 64 bits on the CPU: queries of any
finite size, infinite ones, blocks of values far apart, keys and scales near the limits."""
import math

import pytest
import torch

import _kv8_ref as ref
from test_gpu_kv8 import BF, _check_attention, _fill, _i32, _rand, _starts, kv8  # noqa: F401  (kv8: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("power", [-132, -112, -90, 112, 117, 126])
@pytest.mark.parametrize("m", [1, 60])
def test_queries_of_any_finite_size(kv8, power, m, e4m3):
    """Rows whose largest |q| is near 2^power, subnormal ones among them, against keys near 2^-power: ordinary scores."""
    g = torch.Generator().manual_seed(200 + power)
    n, d, down = 150, 64, min(max(-power, -126), 125)
    draw = lambda *s: torch.randn(*s, generator=g).clamp(-1.9, 1.9).double()  # noqa: E731
    q, k = (draw(m, 4, d) * 2.0 ** power).to(BF), (draw(n, 2, d) * 2.0 ** down).to(BF)
    assert q.isfinite().all() and k.isfinite().all() and float(q.abs().max()) > 0
    cache = kv8.Kv8Cache(1, 2, d, n, format=e4m3)
    kv8.append(cache, k.cuda(), _rand(g, n, 2, d).cuda(), _i32([n]), starts=_starts([n]))
    _, _, _, off = _check_attention(kv8, cache, q, _starts([m]), _i32([n]), scale=2.0 ** (-power - down) / 8)
    assert float(off.max()) < 2.0 ** -8  # (the scores are of ordinary size, so the tolerance means something)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 40), (1, 5000), (60, 150), (60, 5000)])
def test_infinite_queries_whose_scores_are_all_minus_infinity(kv8, m, n, sign):
    """One infinite dim where every key has the other sign: NaN, not zeros; the other rows as without it.  A row that sees
    nothing stays zero."""
    g = torch.Generator().manual_seed(m + n)
    d = 64
    k = _rand(g, n, 2, d)
    k[:, :, 3] = -1.0
    cache = kv8.Kv8Cache(1, 2, d, n)
    kv8.append(cache, k.cuda(), _rand(g, n, 2, d).cuda(), _i32([n]), starts=_starts([n]))
    q, starts, lens, row = _rand(g, m, 4, d), _starts([m]), _i32([n]), m // 2
    fine, fine_lse, _, _ = _check_attention(kv8, cache, q, starts, lens, scale=sign / 8)
    bad = q.clone()
    bad[row, 1, 3] = sign * math.inf
    out, lse = kv8.attention(cache, bad.cuda(), lens, starts=starts, scale=sign / 8)
    assert torch.isnan(out[row, 1]).all() and torch.isnan(lse[row, 1])
    rest = torch.ones(m, 4, dtype=torch.bool)
    rest[row, 1] = False
    # another row's maximum may move a row's base: probabilities in fp16 of values below 6, outputs in bf16, twice
    assert ((out - fine).float().abs()[rest] <= 2 * (2.0 ** -11 + 2.0 ** -8) * 6).all()
    assert ((lse - fine_lse).abs()[rest] <= 1e-5).all()
    weight = kv8.accumulate_weight(cache, bad.cuda(), lse, lens, torch.zeros(1, 2, n, device="cuda"), starts=starts, scale=sign / 8)
    seen = n - m + row + 1
    assert torch.isnan(weight[0, 0, :seen]).all() and torch.isfinite(weight[0, 0, seen:]).all() and torch.isfinite(weight[0, 1]).all()
    none = kv8.attention(cache, bad.cuda(), _i32([0]), starts=starts, scale=sign / 8)
    assert (none[0] == 0).all() and (none[1] == -math.inf).all()


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("power", [16, 20, 26, 40, 60, 100])
@pytest.mark.parametrize("batch,m,n", [(1, 1, 160), (130, 1, 700), (1, 60, 160), (16, 60, 1600)])
def test_blocks_of_large_values_that_a_row_hardly_attends(kv8, batch, m, n, power, e4m3):
    """Blocks of values 2^power times the others', which rows of one sign give weights of e^-40 (2^-58) and rows of the other
    almost all: each row keeps the bits of what it attends."""
    g = torch.Generator().manual_seed(300 + power + n)
    d, t = 64, batch * m
    k, v, q = _rand(g, batch, n, 1, d), _rand(g, batch, n, 1, d).double(), _rand(g, t, 2, d, gain=0.25)
    large = (torch.arange(n) // 32 + torch.arange(batch)[:, None]) % 3 == 1
    k[..., 0] = torch.where(large, -10.0, 0.0)[..., None]
    v[large] *= 2.0 ** power
    q[:, :, 0] = 4.0
    q[::2, 1, 0] = q[1::2, 0, 0] = -4.0
    cache = kv8.Kv8Cache(batch, 1, d, n, format=e4m3)
    lens = [n] * batch
    kv8.append(cache, k.flatten(0, 1).cuda(), v.to(BF).flatten(0, 1).cuda(), _i32(lens), starts=_starts(lens))
    out, lse = kv8.attention(cache, q.cuda(), _i32(lens), starts=_starts([m] * batch), scale=1.0)
    kk, vv = ref.read(cache, n)
    want, wl, mass, terms, _ = ref.attention(q, kk, vv, _starts([m] * batch).cpu(), lens, 1.0, n)
    # the largest product of a probability and its block's largest value
    top = torch.nn.functional.pad(vv.abs().amax(-1), (0, -n % 32)).unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)[:, 0, :n]
    x = (q.double().unflatten(0, (batch, m)).flatten(1, 2) @ kk[:, 0].mT).unflatten(1, (m, 2))
    x = torch.where(torch.arange(n) < (torch.arange(m) + n - m + 1)[:, None, None], x, -math.inf)
    most = (torch.softmax(x, -1) * top[:, None, None]).amax(-1).flatten(0, 1)
    # as in _check_attention, but what fp16 loses below 2^-14 is half of 2^-24 of the row's own largest product; the exponents of
    # two, up to 2^8 in size here, are rounded in f32 (2^-16 of a probability for score, scale and reference)
    off = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -22
    p = 2.0 ** -11 + 2.0 ** -15 + 2 * off[..., None] + 2 * n * 2.0 ** -24
    tol = 2.0 ** -8 * want.abs() + p * mass + n * 2.0 ** -25 * most[..., None]
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert ((lse.cpu().double() - wl).abs() <= off + 2.0 ** -16 + n * 2.0 ** -24 + 2.0 ** -22 * (1 + wl.abs())).all()


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("q_gain,k_gain,scale", [
    (1e-36, 1e36, 0.125), (2.0 ** -49, 2.0 ** -50, 0.9 * 2.0 ** 96), (2.0 ** 20, 2.0 ** -119, -0.9 * 2.0 ** 96),
    (2.0 ** -100, 1.0, 0.9 * 2.0 ** 97), (2.0 ** -120, 2.0 ** 20, 0.9 * 2.0 ** 97), (2.0 ** 50, 2.0 ** 50, 2.0 ** -103),
    (2.0 ** 110, 2.0 ** -113, 1.0)])
@pytest.mark.parametrize("m", [1, 50])
def test_attention_and_weights_near_the_limits(kv8, m, q_gain, k_gain, scale, e4m3):
    """Queries, keys and scale whose product is of ordinary size, each near an end of its range."""
    g = torch.Generator().manual_seed(31)
    n, d = 300, 96
    cache = _fill(kv8, g, [n], 2, d, e4m3, n, gain=k_gain)
    q, starts, lens = _rand(g, m, 4, d, gain=q_gain), _starts([m]), _i32([n])
    out, lse, want, off = _check_attention(kv8, cache, q, starts, lens, scale=scale)
    assert float(off.max()) < 2.0 ** -8  # (ordinary scores: the tolerance means something)
    w = kv8.accumulate_weight(cache, q.cuda(), lse, lens, torch.zeros(1, 2, n, device="cuda"), starts=starts, scale=scale)
    tol = (4 * float(off.max()) + (n + 2 * m) * 2.0 ** -24 + 2.0 ** -20) * want + 1e-30
    assert ((w.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("power", [8, 12, 20, 30, 60, -30])
@pytest.mark.parametrize("step", [40.0, -40.0, 9.0])
@pytest.mark.parametrize("batch,m,n", [(1, 1, 160), (130, 1, 700), (1, 60, 160), (16, 60, 1600)])
def test_equal_scores_of_any_size_over_values_of_many(kv8, batch, m, n, step, power):
    """Every key the same, scores near 2^power (or -2^30): a plain average, whatever the blocks' scales of values are."""
    g = torch.Generator().manual_seed(400 + n)
    d = 64
    block = torch.arange(n) // 32
    v = _rand(g, batch, n, 1, d).double() * torch.exp2(step * (block % 3))[:, None, None]
    k = torch.ones(batch, n, 1, d, dtype=BF)
    q = torch.ones(batch * m, 2, d, dtype=BF)
    scale = 2.0 ** (abs(power) - 6) * (1 if power > 0 else -1)
    cache, lens = kv8.Kv8Cache(batch, 1, d, n), [n] * batch
    kv8.append(cache, k.flatten(0, 1).cuda(), v.to(BF).flatten(0, 1).cuda(), _i32(lens), starts=_starts(lens))
    out, lse = kv8.attention(cache, q.cuda(), _i32(lens), starts=_starts([m] * batch), scale=scale)
    _, vv = ref.read(cache, n)
    seen = torch.arange(m) + n - m + 1
    cut = (torch.arange(n) < seen[:, None]).double() / seen[:, None]  # [m, n]
    want, mass = cut @ vv[:, 0], cut @ vv[:, 0].abs()               # [batch, m, d]
    most = vv[:, 0].abs().amax((1, 2))[:, None, None] / seen[:, None]
    got = out.cpu().double().unflatten(0, (batch, m))
    # the scores are the same bits, so only fp16's and bf16's half steps, sums of n in f32 and the exponents' 2^-14 (2^-15 of scores below 2^10)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13 + 2 * n * 2.0 ** -24) * mass + n * 2.0 ** -25 * most
    assert ((got - want[:, :, None]).abs() <= tol[:, :, None]).all()
    at = scale * 64 * float(ref.read(cache, 1)[0][0, 0, 0, 0])
    wl = at + torch.log(seen.double())[:, None]
    assert ((lse.cpu().double().unflatten(0, (batch, m)) - wl).abs() <= (d + 8) * 2.0 ** -24 * abs(at) + n * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(at))).all()


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("batch,m,n", [(1, 1, 33), (1, 1, 160), (1, 2, 5000), (3, 1, 40000), (1, 60, 160), (1, 60, 5000), (1, 600, 4000)])
def test_values_near_the_largest(kv8, batch, m, n, e4m3):
    """Values up to 2^127: their averages are finite, however many waves and parts they are joined from."""
    g = torch.Generator().manual_seed(500 + n)
    d, lens = 64, [n] * batch
    k = _rand(g, batch * n, 1, d)
    v = ((torch.rand(batch * n, 1, d, generator=g) - 0.25) * 2.0 ** 127).to(BF)
    cache = kv8.Kv8Cache(batch, 1, d, n, format=e4m3)
    kv8.append(cache, k.cuda(), v.cuda(), _i32(lens), starts=_starts(lens))
    q = _rand(g, batch * m, 2, d, gain=0.5)
    out, lse, _, _ = _check_attention(kv8, cache, q, _starts([m] * batch), _i32(lens))
    assert out.isfinite().all() and lse.isfinite().all()
