"""CPU checks of the paged cache's entry points: what they refuse before any launch, their workspace sizes, and the Python binding's
own checks (no GPU work here)."""
import ctypes
import math

import pytest
import torch

import _paged_ref as ref


@pytest.fixture(scope="module")
def kq():
    import os

    import kriya_q4

    if not os.path.exists(kriya_q4.LIB_PATH):
        kriya_q4.build()
    kriya_q4.lib()
    return kriya_q4


def _cache(**kw):
    from kriya_q4 import paged

    return paged.kr_paged_cache(*dict(dict(k=0x10000, v=0x20000, layers=2, pages=10, page=16, kv_heads=2, head_dim=64), **kw).values())


def _step(**kw):
    from kriya_q4 import paged

    return paged.kr_paged_step(*dict(dict(table=0x30000, max_pages=6, batch=2, starts=None, lengths=0x40000), **kw).values())


X, WS = 0x70000, 1 << 30


def _append(L, cache, step, layer=0, norm=None, rope=None, k=X, v=X, kvs=128, q=None, qo=None, qs=0, qh=0, tokens=2):
    return L.kr_paged_append(cache, layer, step, norm, rope, k, v, kvs, q, qo, qs, qh, tokens, None)


def _read(L, cache, step, layer=0, first=None, count=10, k=X, v=X, dtype=0):
    return L.kr_paged_read(cache, layer, step, first, count, k, v, dtype, None)


def _attend(L, cache, step, layer=0, q=X, qs=256, qh=4, tokens=2, mask=None, words=0, scale=0.125, out=0xA0000, lse=0xB0000,
            ws=0xC0000, wb=WS):
    return L.kr_paged_attention(cache, layer, step, q, qs, qh, tokens, mask, words, scale, out, lse, ws, wb, None)


def _commit(L, cache, step, drafted=X, parents=X, targets=X, tokens=2, most=4, path=X, counts=X, nxt=X, lengths=X):
    return L.kr_paged_commit(cache, step, drafted, parents, targets, tokens, most, path, counts, nxt, lengths, None)


CALLS = [_append, _read, _attend, _commit]


@pytest.mark.parametrize("change,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(k=0x10008), -3), (dict(v=0x20002), -3), (dict(kv_heads=0), -2),
    (dict(kv_heads=65536), -2), (dict(pages=0), -2), (dict(pages=1 << 31), -2), (dict(layers=0), -2), (dict(layers=65536), -2),
    (dict(page=0), -6), (dict(page=8), -6), (dict(page=48), -6), (dict(page=8192), -6), (dict(head_dim=80), -6), (dict(head_dim=0), -6)])
def test_every_entry_point_refuses_a_bad_cache(kq, change, code):
    L = kq.lib()
    for call in CALLS:
        assert call(L, ctypes.byref(_cache(**change)), ctypes.byref(_step())) == code
        assert call(L, None, ctypes.byref(_step())) == kq.KR_E_INVALID


@pytest.mark.parametrize("change,code", [
    (dict(table=None), -1), (dict(table=0x30002), -3), (dict(max_pages=0), -2), (dict(max_pages=(1 << 26) + 1), -2),
    (dict(batch=65536), -2), (dict(lengths=None), -1), (dict(lengths=0x40001), -3), (dict(starts=0x50002), -3)])
def test_every_entry_point_refuses_a_bad_step(kq, change, code):
    L = kq.lib()
    for call in CALLS:
        assert call(L, ctypes.byref(_cache()), ctypes.byref(_step(**change))) == code
        assert call(L, ctypes.byref(_cache()), None) == kq.KR_E_INVALID


def test_layers_and_token_counts(kq):
    L, c, s = kq.lib(), ctypes.byref(_cache()), ctypes.byref(_step())
    for call in (_append, _read, _attend):
        assert call(L, c, s, layer=2) == kq.KR_E_SHAPE
    for call in (_append, _attend, _commit):
        assert call(L, c, s, tokens=3) == kq.KR_E_SHAPE  # without starts: one token a sequence
    none = ctypes.byref(_step(batch=0, table=None, lengths=None))
    assert _append(L, c, s, tokens=0) == 0 and _attend(L, c, s, tokens=0, q=None, out=None, ws=None, wb=0) == 0
    assert _read(L, c, s, count=0) == 0 and _read(L, c, s, k=None, v=None) == 0
    for call in CALLS:
        assert call(L, c, none) == 0  # nothing to do, nothing launched


def test_append_refusals(kq):
    from kriya_q4.paged import kr_head_norm
    from kriya_q4.rope import kr_rope

    L, c, s = kq.lib(), ctypes.byref(_cache()), ctypes.byref(_step())
    rope = lambda **kw: ctypes.byref(kr_rope(*dict(dict(cos_sin=0x90000, positions=X, rows=10, rotary_dim=64, layout=0, inverse=0), **kw).values()))  # noqa: E731
    norm = lambda q=X, k=X, eps=1e-6: ctypes.byref(kr_head_norm(q, k, eps))  # noqa: E731
    call = lambda **kw: _append(L, c, s, **kw)  # noqa: E731
    assert call(k=None) == kq.KR_E_INVALID and call(v=None) == kq.KR_E_INVALID
    assert call(k=X + 8) == kq.KR_E_ALIGN and call(v=X + 8) == kq.KR_E_ALIGN
    assert call(kvs=127) == kq.KR_E_SHAPE and call(kvs=132) == kq.KR_E_SHAPE and call(kvs=120) == kq.KR_E_SHAPE
    assert call(q=X, qo=X, qs=256, qh=4) == kq.KR_E_INVALID  # q without norm and rope
    for more in (dict(rope=rope()), dict(norm=norm())):
        assert call(q=X, qo=None, qs=256, qh=4, **more) == kq.KR_E_INVALID
        assert call(q=X, qo=X, qs=255, qh=4, **more) == kq.KR_E_SHAPE and call(q=X, qo=X, qs=256, qh=0, **more) == kq.KR_E_SHAPE
        assert call(q=X + 4, qo=X, qs=256, qh=4, **more) == kq.KR_E_ALIGN and call(q=X, qo=X + 4, qs=256, qh=4, **more) == kq.KR_E_ALIGN
    assert call(norm=norm(q=X + 1)) == kq.KR_E_ALIGN and call(norm=norm(k=X + 1)) == kq.KR_E_ALIGN
    assert call(norm=norm(eps=-1.0)) == kq.KR_E_INVALID and call(norm=norm(eps=math.nan)) == kq.KR_E_INVALID
    assert call(norm=norm(eps=math.inf)) == kq.KR_E_INVALID
    assert call(rope=rope(inverse=1)) == kq.KR_E_INVALID and call(rope=rope(layout=2)) == kq.KR_E_INVALID
    assert call(rope=rope(rotary_dim=66)) == kq.KR_E_SHAPE and call(rope=rope(rotary_dim=63)) == kq.KR_E_SHAPE
    assert call(rope=rope(positions=None)) == kq.KR_E_INVALID and call(rope=rope(cos_sin=0x90004)) == kq.KR_E_ALIGN
    assert call(rope=rope(rows=0)) == kq.KR_E_SHAPE
    wide = ctypes.byref(_step(starts=0x50000))
    assert _append(L, c, wide, tokens=1 << 30, rope=rope(), q=X, qo=X, qs=256, qh=4) == kq.KR_E_SHAPE


def test_attention_refusals(kq):
    L, c, s = kq.lib(), ctypes.byref(_cache()), ctypes.byref(_step())
    call = lambda **kw: _attend(L, c, s, **kw)  # noqa: E731
    assert call(q=None) == kq.KR_E_INVALID and call(out=None) == kq.KR_E_INVALID
    assert call(q=X + 8) == kq.KR_E_ALIGN and call(out=0xA0008) == kq.KR_E_ALIGN and call(lse=0xB0002) == kq.KR_E_ALIGN
    assert call(qh=3) == kq.KR_E_SHAPE and call(qh=0) == kq.KR_E_SHAPE
    assert call(qs=248) == kq.KR_E_SHAPE and call(qs=260) == kq.KR_E_SHAPE
    assert call(scale=math.inf) == kq.KR_E_INVALID and call(scale=math.nan) == kq.KR_E_INVALID and call(scale=2.0 ** 100) == kq.KR_E_INVALID
    assert call(mask=X, words=0) == kq.KR_E_SHAPE and call(mask=X, words=(1 << 20) + 1) == kq.KR_E_SHAPE and call(mask=X + 2, words=1) == kq.KR_E_ALIGN
    need = L.kr_paged_attention_workspace_bytes(c, s, 4, 2)
    assert need > 0 and need % 256 == 0
    assert call(ws=None) == kq.KR_E_WORKSPACE and call(wb=need - 1) == kq.KR_E_WORKSPACE and call(ws=0xC0008) == kq.KR_E_ALIGN
    assert _attend(L, c, ctypes.byref(_step(starts=0x50000)), tokens=1 << 30) == kq.KR_E_SHAPE


def test_plan_and_commit_refusals(kq):
    L, c, s = kq.lib(), ctypes.byref(_cache()), ctypes.byref(_step())

    def plan(parents=X, tokens=2, starts=None, lengths=X, batch=2, words=1, mask=X, positions=X):
        return L.kr_tree_plan(parents, tokens, starts, lengths, batch, words, mask, positions, None)
    assert plan(words=0) == kq.KR_E_SHAPE and plan(words=129) == kq.KR_E_SHAPE and plan(batch=65536) == kq.KR_E_SHAPE
    assert plan(tokens=3) == kq.KR_E_SHAPE and plan(lengths=None) == kq.KR_E_INVALID and plan(lengths=X + 2) == kq.KR_E_ALIGN
    for name in ("parents", "mask", "positions"):
        assert plan(**{name: None}) == kq.KR_E_INVALID and plan(**{name: X + 2}) == kq.KR_E_ALIGN
    assert plan(tokens=0, parents=None) == 0 and plan(batch=0) == 0
    for name in ("drafted", "parents", "targets", "path", "counts", "nxt", "lengths"):
        assert _commit(L, c, s, **{name: None}) == kq.KR_E_INVALID and _commit(L, c, s, **{name: X + 2}) == kq.KR_E_ALIGN
    assert _commit(L, c, s, most=0) == kq.KR_E_SHAPE and _commit(L, c, s, most=4097) == kq.KR_E_SHAPE
    assert _commit(L, c, s, lengths=0x40000) == kq.KR_E_INVALID  # the step's own


def test_written_memory_lies_apart(kq):
    """Outputs over inputs or one another: refused, by whole ranges (2 sequences, 2 tokens of 4 heads of 64)."""
    L = kq.lib()
    cache, step = ctypes.byref(_cache()), ctypes.byref(_step())
    for change in (dict(out=X), dict(out=X + 1008), dict(out=X - 1008), dict(lse=X + 1020), dict(lse=0xA0000 + 1020), dict(ws=X - 16),
                   dict(ws=0xB0000), dict(mask=0xA0000 + 1020, words=1), dict(mask=0xB0000, words=2)):
        assert _attend(L, cache, step, **change) == kq.KR_E_INVALID, change
    apart = dict(drafted=0x80000, parents=0x81000, targets=0x82000, path=0x83000, counts=0x84000, nxt=0x85000, lengths=0x86000)
    for name, size in (("path", 32), ("counts", 8), ("nxt", 8), ("lengths", 8)):
        for at in (0x80000, 0x81004, 0x82000, 0x40000, 0x30000 + 44):  # the inputs, the step's lengths, the table's last
            assert _commit(L, cache, step, **dict(apart, **{name: at})) == kq.KR_E_INVALID, (name, hex(at))
        for other in apart:
            if other != name:
                assert _commit(L, cache, step, **dict(apart, **{other: apart[name] + size - 4})) == kq.KR_E_INVALID, (name, other)
    plan = lambda mask, positions: L.kr_tree_plan(0x80000, 10, 0x81000, 0x82000, 2, 2, mask, positions, None)  # noqa: E731
    for mask, positions in ((0x80000, 0x90000), (0x90000, 0x80000 + 36), (0x90000, 0x90000 + 76), (0x81000 + 8, 0x90000), (0x90000, 0x82004)):
        assert plan(mask, positions) == kq.KR_E_INVALID


def test_workspace_is_bounded(kq):
    L = kq.lib()
    assert L.kr_paged_attention_workspace_bytes(None, ctypes.byref(_step()), 4, 2) == 0
    assert L.kr_paged_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(_step()), 3, 2) == 0
    for b, h, g, d, t in ((1, 1, 1, 64, 1), (1, 2, 8, 128, 1), (64, 8, 4, 128, 64), (16, 2, 8, 256, 16), (4, 2, 5, 256, 600),
                          (1, 2, 8, 128, 3907), (8, 8, 16, 64, 8000)):
        need = L.kr_paged_attention_workspace_bytes(ctypes.byref(_cache(kv_heads=h, head_dim=d)), ctypes.byref(_step(batch=b, max_pages=1000)), g * h, t)
        assert need % 256 == 0 and need < 1 << 28, (b, h, g, d, t, need)


def test_binding_refuses_what_is_not_on_the_gpu():
    from kriya_q4 import paged

    k = torch.zeros(1, 2, 1, 1, 16 * 64, dtype=torch.bfloat16)
    for bad in (k, k[0], k.float(), torch.zeros(1, 2, 1, 1, 100, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            paged.PagedCache.wrap(bad, bad)
    with pytest.raises(ValueError):
        paged.PagedCache(1, 2, 24, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        paged.Step(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        paged.tree_plan(torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), nodes=3)


def test_reference_layout_is_one_to_one():
    for d in (64, 96, 128, 192, 256):
        for at in (ref.key_at, ref.value_at):
            assert sorted(at(r, x) for r in range(16) for x in range(d)) == list(range(16 * d))


def test_reference_plan_and_path():
    rows, positions = ref.plan([-1, 0, 0, 1, 7, 3], 10, 1)
    assert rows == [[1], [3], [5], [11], [16], [43]] and positions == [4, 5, 5, 6, 4, 7]
    assert ref.path([5, 6, 6, 7], [-1, 0, 0, 2], [6, 7, 7, 9], 4) == [0, 1] and ref.path([], [], [], 3) == []
