"""CPU checks of the rotary and 8-bit cache entry points: what they refuse before any launch, their workspace sizes, and
the Python binding's own checks (no GPU work here)."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def kq():
    import os

    import kriya_q4

    if not os.path.exists(kriya_q4.LIB_PATH):
        kriya_q4.build()
    kriya_q4.lib()
    return kriya_q4


def _cache(**kw):
    from kriya_q4 import kv8

    f = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, k_open=0x50000, v_open=0x60000, batch=2, kv_heads=2,
             head_dim=64, max_ctx=100, format=0)
    f.update(kw)
    return kv8.kr_kv8_cache(*f.values())


BAD_CACHES = [(dict(k=None), -1), (dict(v_open=None), -1), (dict(k=0x10008), -3), (dict(k_open=0x50002), -3),
              (dict(v_scale=0x40002), -3), (dict(kv_heads=0), -2), (dict(max_ctx=0), -2), (dict(max_ctx=(1 << 30) + 1), -2),
              (dict(head_dim=80), -6), (dict(head_dim=0), -6), (dict(format=2), -1), (dict(batch=65536), -2)]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_every_entry_point_refuses_a_bad_cache(kq, change, code):
    L = kq.lib()
    good, bad = ctypes.byref(_cache()), ctypes.byref(_cache(**change))
    x, n = 0x70000, 0x80000
    assert L.kr_kv8_append(bad, None, x, x, 128, None, None, 0, 0, 2, None, n, None) == code
    assert L.kr_kv8_dequant(bad, n, None, 10, x, x, 0, None) == code
    assert L.kr_kv8_attention(bad, x, 256, 4, 2, None, n, 0.125, x, None, x, 1 << 30, None) == code
    assert L.kr_kv8_accumulate_weight(bad, x, 256, 4, 2, None, n, 0.125, x, 1.0, x, x, 1 << 30, None) == code
    assert L.kr_kv8_evict(bad, n, x, 10, 1, 1, good, x + 64, x, None, None) == code
    assert L.kr_kv8_evict(good, n, x, 10, 1, 1, bad, x + 64, x, None, None) == code
    assert L.kr_kv8_append(None, None, x, x, 128, None, None, 0, 0, 2, None, n, None) == kq.KR_E_INVALID


def test_append_refusals(kq):
    from kriya_q4.rope import kr_rope

    L, c = kq.lib(), ctypes.byref(_cache())
    k, n, cs = 0x70000, 0x80000, 0x90000
    rope = lambda **kw: ctypes.byref(kr_rope(*dict(dict(cos_sin=cs, positions=n, rows=10, rotary_dim=64, layout=0, inverse=0), **kw).values()))  # noqa: E731
    ok = dict(rope=None, k=k, v=k, kvs=128, q=None, qo=None, qs=0, qh=0, tokens=2, starts=None, lengths=n)

    def call(**kw):
        a = dict(ok, **kw)
        return L.kr_kv8_append(c, a["rope"], a["k"], a["v"], a["kvs"], a["q"], a["qo"], a["qs"], a["qh"], a["tokens"], a["starts"], a["lengths"], None)
    assert call(k=None) == kq.KR_E_INVALID
    assert call(v=k + 8) == kq.KR_E_ALIGN
    assert call(kvs=127) == kq.KR_E_SHAPE and call(kvs=132) == kq.KR_E_SHAPE and call(kvs=120) == kq.KR_E_SHAPE
    assert call(lengths=None) == kq.KR_E_INVALID
    assert call(tokens=3) == kq.KR_E_SHAPE          # without starts: one token a sequence
    assert call(q=k, qo=k, qs=256, qh=4) == kq.KR_E_INVALID  # q without rope
    assert call(rope=rope(inverse=1)) == kq.KR_E_INVALID
    assert call(rope=rope(rotary_dim=66)) == kq.KR_E_SHAPE and call(rope=rope(rotary_dim=63)) == kq.KR_E_SHAPE
    assert call(rope=rope(layout=2)) == kq.KR_E_INVALID and call(rope=rope(positions=None)) == kq.KR_E_INVALID
    assert call(rope=rope(cos_sin=cs + 4)) == kq.KR_E_ALIGN
    assert call(rope=rope(), q=k, qo=None, qs=256, qh=4) == kq.KR_E_INVALID
    assert call(rope=rope(), q=k, qo=k, qs=255, qh=4) == kq.KR_E_SHAPE
    assert call(rope=rope(), q=k + 4, qo=k, qs=256, qh=4) == kq.KR_E_ALIGN
    assert call(tokens=0, k=None, lengths=None) == 0  # nothing to append, nothing launched


def test_attention_and_weight_refusals(kq):
    L, c = kq.lib(), _cache()
    cr = ctypes.byref(c)
    q, n, big = 0x70000, 0x80000, 1 << 30
    need = L.kr_kv8_attention_workspace_bytes(cr, 4, 2)
    assert need % 256 == 0

    def att(q=q, qs=256, qh=4, t=2, st=None, n=n, sc=0.125, out=0xA0000, lse=0xB0000, ws=0xC0000, wb=big):
        return L.kr_kv8_attention(cr, q, qs, qh, t, st, n, sc, out, lse, ws, wb, None)

    def wei(q=q, qs=256, qh=4, t=2, st=None, n=n, sc=0.125, lse=0xB0000, de=1.0, w=0xD0000, ws=0xE0000, wb=big):
        return L.kr_kv8_accumulate_weight(cr, q, qs, qh, t, st, n, sc, lse, de, w, ws, wb, None)
    for f in (att, wei):
        assert f(q=None) == kq.KR_E_INVALID and f(q=q + 8) == kq.KR_E_ALIGN
        assert f(qh=3) == kq.KR_E_SHAPE and f(qh=0) == kq.KR_E_SHAPE
        assert f(qs=248) == kq.KR_E_SHAPE and f(qs=260) == kq.KR_E_SHAPE
        assert f(t=3) == kq.KR_E_SHAPE and f(n=None) == kq.KR_E_INVALID and f(n=n + 2) == kq.KR_E_ALIGN
        assert f(sc=math.inf) == kq.KR_E_INVALID and f(sc=math.nan) == kq.KR_E_INVALID
        assert f(t=1 << 30, st=n) == kq.KR_E_SHAPE
        assert f(t=0, q=None, n=None) == 0
    assert att(out=None) == kq.KR_E_INVALID and att(out=0xA0008) == kq.KR_E_ALIGN and att(lse=0xB0002) == kq.KR_E_ALIGN
    assert att(ws=0xC0008) == kq.KR_E_ALIGN
    if need:
        assert att(ws=None) == kq.KR_E_WORKSPACE and att(wb=need - 1) == kq.KR_E_WORKSPACE
    assert wei(lse=None) == kq.KR_E_INVALID and wei(w=None) == kq.KR_E_INVALID and wei(w=0xD0001) == kq.KR_E_ALIGN
    assert wei(de=math.inf) == kq.KR_E_INVALID and wei(ws=0xE0008) == kq.KR_E_ALIGN
    assert L.kr_kv8_weight_workspace_bytes(cr, 4, 2) == 0
    need = L.kr_kv8_weight_workspace_bytes(cr, 4, 1000)
    assert need >= 2 * 2 * 100 * 4 and need % 256 == 0
    assert wei(t=1000, st=n, ws=None) == kq.KR_E_WORKSPACE and wei(t=1000, st=n, wb=need - 1) == kq.KR_E_WORKSPACE


def test_attention_workspace_grows_with_the_step_and_is_bounded(kq):
    L = kq.lib()
    assert L.kr_kv8_attention_workspace_bytes(None, 4, 2) == 0
    assert L.kr_kv8_attention_workspace_bytes(ctypes.byref(_cache()), 3, 2) == 0
    for b, h, g, d, t in ((1, 1, 1, 64, 1), (1, 2, 8, 128, 1), (64, 8, 4, 128, 64), (16, 2, 8, 256, 16), (4, 2, 5, 256, 600),
                          (1, 2, 8, 128, 3907), (8, 8, 16, 64, 8000)):
        need = L.kr_kv8_attention_workspace_bytes(ctypes.byref(_cache(batch=b, kv_heads=h, head_dim=d)), g * h, t)
        assert need % 256 == 0 and need < 1 << 28, (b, h, g, d, t, need)


def test_evict_and_dequant_refusals(kq):
    L = kq.lib()
    c, n, w, w2, kept = _cache(), 0x80000, 0x90000, 0xA0000, 0xB0000
    to = dict(k=0x110000, v=0x120000, k_scale=0x130000, v_scale=0x140000, k_open=0x150000, v_open=0x160000, max_ctx=50)

    def ev(c=c, n=n, w=w, budget=20, sink=4, recent=8, to=_cache(**to), w2=w2, kept=kept, n2=None):
        return L.kr_kv8_evict(ctypes.byref(c), n, w, budget, sink, recent, ctypes.byref(to), w2, kept, n2, None)
    assert ev(budget=0, sink=0, recent=0) == kq.KR_E_SHAPE and ev(budget=51) == kq.KR_E_SHAPE
    assert ev(sink=13) == kq.KR_E_SHAPE and ev(sink=0xFFFFFFFF) == kq.KR_E_SHAPE
    for name in ("k", "v", "k_scale", "v_scale", "k_open", "v_open"):  # shared with the source
        assert ev(to=_cache(**dict(to, **{name: getattr(c, name)}))) == kq.KR_E_INVALID
    assert ev(w2=w) == kq.KR_E_INVALID and ev(n2=n) == kq.KR_E_INVALID
    assert ev(kept=None) == kq.KR_E_INVALID and ev(n=None) == kq.KR_E_INVALID and ev(kept=kept + 1) == kq.KR_E_ALIGN
    for change in (dict(batch=3), dict(kv_heads=4), dict(head_dim=128), dict(format=1)):
        assert ev(to=_cache(**dict(to, **change))) == kq.KR_E_SHAPE
    cr = ctypes.byref(c)
    assert L.kr_kv8_dequant(cr, n, None, 5, 0x70008, 0x70000, 0, None) == kq.KR_E_ALIGN
    assert L.kr_kv8_dequant(cr, n, None, 5, 0x70000, 0x70000, 7, None) == kq.KR_E_INVALID
    assert L.kr_kv8_dequant(cr, None, None, 5, 0x70000, 0x70000, 0, None) == kq.KR_E_INVALID
    assert L.kr_kv8_dequant(cr, n, None, (1 << 30) + 1, 0x70000, 0x70000, 0, None) == kq.KR_E_SHAPE
    assert L.kr_kv8_dequant(cr, n, None, 0, None, None, 0, None) == 0


def test_rope_refusals(kq):
    from kriya_q4.rope import kr_rope, kr_rope_scaling

    L = kq.lib()
    out = 0x10000

    def tab(out=out, first=0, count=8, r=64, theta=1e4, z=None):
        return L.kr_rope_table(out, first, count, r, theta, ctypes.byref(z) if z else None, None)
    assert tab(r=0) == kq.KR_E_SHAPE and tab(r=63) == kq.KR_E_SHAPE and tab(r=258) == kq.KR_E_SHAPE
    assert tab(theta=0.0) == kq.KR_E_INVALID and tab(theta=math.inf) == kq.KR_E_INVALID and tab(theta=math.nan) == kq.KR_E_INVALID
    assert tab(out=None) == kq.KR_E_INVALID and tab(out=out + 4) == kq.KR_E_ALIGN
    assert tab(first=0xFFFFFFFF, count=2) == kq.KR_E_SHAPE and tab(count=0, out=None) == 0
    assert tab(z=kr_rope_scaling(4, 2.0, 1.0, 0.0, 1.0, 1.0)) == kq.KR_E_INVALID
    assert tab(z=kr_rope_scaling(1, 0.0, 1.0, 0.0, 1.0, 1.0)) == kq.KR_E_INVALID
    assert tab(z=kr_rope_scaling(2, 2.0, 1.0, 0.0, 1.0, 1.0), r=2) == kq.KR_E_SHAPE
    assert tab(z=kr_rope_scaling(3, 2.0, 0.0, 1.0, 32.0, 1.0)) == kq.KR_E_INVALID
    assert tab(z=kr_rope_scaling(3, 2.0, 4096.0, 32.0, 1.0, 1.0)) == kq.KR_E_INVALID
    assert tab(z=kr_rope_scaling(0, 1.0, 0.0, 0.0, 0.0, math.inf)) == kq.KR_E_INVALID
    base = dict(cos_sin=0x20000, positions=0x30000, rows=10, rotary_dim=64, layout=0, inverse=0)

    def app(x=0x40000, xs=256, y=0x50000, ys=256, dt=0, t=3, h=2, d=128, **kw):
        r = kr_rope(*dict(base, **kw).values())
        return L.kr_rope_apply(ctypes.byref(r), x, xs, y, ys, dt, t, h, d, None)
    assert app(x=None) == kq.KR_E_INVALID and app(y=0x50001) == kq.KR_E_ALIGN and app(dt=1, x=0x40002) == kq.KR_E_ALIGN
    assert app(xs=255) == kq.KR_E_SHAPE and app(y=0x40000, ys=300) == kq.KR_E_SHAPE
    assert app(dt=2) == kq.KR_E_INVALID and app(h=0) == kq.KR_E_SHAPE and app(d=1) == kq.KR_E_SHAPE
    assert app(rotary_dim=130) == kq.KR_E_SHAPE and app(layout=5) == kq.KR_E_INVALID and app(inverse=2) == kq.KR_E_INVALID
    assert app(t=0, x=None) == 0
    assert L.kr_rope_apply(None, 1, 1, 1, 1, 0, 1, 1, 2, None) == kq.KR_E_INVALID


def test_calls_too_large_for_a_launch_and_tables_without_rows(kq):
    from kriya_q4.rope import kr_rope, kr_rope_scaling

    L, n, x, big = kq.lib(), 0x80000, 0x70000, 1 << 62
    wide = _cache(batch=65535, kv_heads=65535)
    empty = kr_rope(0x20000, 0x30000, 0, 64, 0, 0)
    full = kr_rope(0x20000, 0x30000, 10, 64, 0, 0)
    assert L.kr_rope_apply(ctypes.byref(empty), x, 256, x, 256, 0, 3, 2, 128, None) == kq.KR_E_SHAPE
    assert L.kr_kv8_append(ctypes.byref(_cache()), ctypes.byref(empty), x, x, 128, None, None, 0, 0, 2, None, n, None) == kq.KR_E_SHAPE
    assert L.kr_rope_apply(ctypes.byref(full), x, 256, x, 256, 0, 1 << 24, 2, 128, None) == kq.KR_E_SHAPE
    assert L.kr_rope_table(x, 0, 1 << 26, 128, 1e4, None, None) == kq.KR_E_SHAPE
    assert L.kr_rope_table(x, 0, 8, 128, 1e4, ctypes.byref(kr_rope_scaling(0, 1.0, 0.0, 0.0, 0.0, 1e39)), None) == kq.KR_E_INVALID
    assert L.kr_kv8_append(ctypes.byref(wide), None, x, x, 65535 * 64, None, None, 0, 0, 65535, None, n, None) == kq.KR_E_SHAPE
    assert L.kr_kv8_append(ctypes.byref(_cache()), None, x, x, 128, None, None, 0, 0, 1 << 25, n, n, None) == kq.KR_E_SHAPE
    many = _cache(batch=60000, kv_heads=300)  # 65 rows a sequence and head, a workgroup each at least
    assert L.kr_kv8_attention(ctypes.byref(many), x, 65 * 300 * 64, 65 * 300, 60000, n, n, 0.125, x, x, x, big, None) == kq.KR_E_SHAPE
    long = dict(max_ctx=1 << 30)
    to = _cache(k=0x110000, v=0x120000, k_scale=0x130000, v_scale=0x140000, k_open=0x150000, v_open=0x160000, **long)
    assert L.kr_kv8_evict(ctypes.byref(_cache(**long)), n, x, 1 << 30, 0, 0, ctypes.byref(to), x + 64, x, None, None) == kq.KR_E_SHAPE


def test_python_checks_name_the_tensor(kq):
    from kriya_q4 import kv8, rope

    with pytest.raises(ValueError, match="on the GPU"):
        kv8.Kv8Cache(1, 1, 64, 40, device="cpu")
    with pytest.raises(ValueError, match="must be on the same GPU|on the GPU"):
        rope.apply(torch.zeros(2, 1, 64), torch.zeros(4, 32, 2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="scaling kind"):
        rope.Scaling("cubic")._c()
    assert rope.Scaling("parts", 4.0, 4096)._c().gain == pytest.approx(0.1 * math.log(4.0) + 1.0)
    assert rope.Scaling("linear", 4.0)._c().gain == 1.0
