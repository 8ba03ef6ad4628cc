"""CPU checks of the paged cache's entry points at the ends of their sizes, and of what their arguments may share (no GPU work here)."""
import ctypes

import pytest

from test_paged_checks import _cache, _step, kq  # noqa: F401  (kq: the fixture)


def _workspace(L, q_heads, tokens, cache=None, step=None):
    return L.kr_paged_attention_workspace_bytes(ctypes.byref(_cache(**(cache or {}))), ctypes.byref(_step(**(step or {}))), q_heads, tokens)


# ---- the workspace of attention

@pytest.mark.parametrize("q_heads,tokens,step", [(4, 2, {}), (16, 200, dict(batch=1, max_pages=100000))], ids=["few", "many"])
def test_no_workspace_for_what_the_call_refuses(kq, q_heads, tokens, step):
    """Sizes that attention refuses give 0, and no arithmetic on them (a head_dim of 0 was divided by)."""
    L = kq.lib()
    assert _workspace(L, q_heads, tokens, {}, step) > 0
    for cache in (dict(head_dim=0), dict(head_dim=80), dict(head_dim=512), dict(page=0), dict(page=48), dict(page=8192), dict(kv_heads=0),
                  dict(kv_heads=65536), dict(pages=0), dict(pages=1 << 31), dict(layers=0)):
        assert _workspace(L, q_heads, tokens, cache, step) == 0, cache
    for change in (dict(max_pages=0), dict(max_pages=(1 << 26) + 1), dict(max_pages=1 << 28), dict(batch=65536)):  # 2^28 pages of 16: 2^32 slots
        assert _workspace(L, q_heads, tokens, {}, dict(step, **change)) == 0, change
    assert _workspace(L, 0, tokens, {}, step) == 0 and _workspace(L, 3, tokens, {}, step) == 0
    assert _workspace(L, 65536, tokens, {}, step) == 0 and _workspace(L, q_heads, 1 << 30, {}, step) == 0
    assert L.kr_paged_attention_workspace_bytes(None, None, q_heads, tokens) == 0


@pytest.mark.parametrize("d,tiles", [(64, 8388607), (128, 8388607), (192, 16777215), (256, 16777215)])
def test_launches_of_too_many_threads_are_refused(kq, d, tiles):
    """A launch has fewer than 2^32 threads: tiles of 128 rows by 512 threads up to a head_dim of 128, by 256 above.  (The call with
    sizes that fit goes on to its pointers.)"""
    L, c = kq.lib(), ctypes.byref(_cache(kv_heads=1, head_dim=d))
    s = ctypes.byref(_step(batch=1, starts=0x50000))

    def call(tokens):
        return L.kr_paged_attention(c, 0, s, None, d, 1, tokens, None, 0, 0.125, None, None, None, 0, None)
    rows = 128 * (tiles - 1)  # and one tile that is not full
    assert call(rows) == call(rows + 127) == kq.KR_E_INVALID
    if rows + 128 < 1 << 31:
        assert call(rows + 128) == kq.KR_E_SHAPE


@pytest.mark.parametrize("batch", [64, 600, 1100, 4096, 16384, 65535])
@pytest.mark.parametrize("kv,group,d", [(1, 4, 64), (8, 4, 128), (2, 8, 256), (8, 16, 64)])
def test_the_workspace_of_a_large_batch_is_bounded(kq, batch, kv, group, d):
    """One token each: no more parts have a place than a launch may split its tiles into (at most 1536 a kv head), however many
    sequences there are."""
    most = 1536 * kv * 16 * (d + 2) * 4 + 512
    for starts in (None, 0x50000):
        assert 0 < _workspace(kq.lib(), kv * group, batch, dict(kv_heads=kv, head_dim=d), dict(batch=batch, max_pages=1000, starts=starts)) <= most


# ---- memory that is written and read

Q, K, V, QO = 0x100000, 0x200000, 0x300000, 0x400000


def _append(L, layer=0, tokens=20, k=K, v=V, kvs=128, q=Q, qo=QO, qs=256, norm=None, rope=None, **step):
    """20 tokens of 4 and 2 heads of 64; a layer of 10 pages is 0xA000 bytes at 0x1000000 and 0x2000000."""
    from kriya_q4.paged import kr_head_norm

    norm = norm or kr_head_norm(0x500000, 0x500100, 1e-6)
    step = _step(**dict(dict(starts=0x600000, lengths=0x601000, table=0x602000), **step))
    cache = _cache(k=0x1000000, v=0x2000000)
    return L.kr_paged_append(ctypes.byref(cache), layer, ctypes.byref(step), ctypes.byref(norm), None if rope is None else ctypes.byref(rope), k, v,
                             kvs, q, qo, qs, 4, tokens, None)


def test_append_refuses_what_it_writes_and_reads(kq):
    """q_out over rows of q other than its own, over k, v, a weight, the table ..; the layer's pages over any of them."""
    from kriya_q4.paged import kr_head_norm
    from kriya_q4.rope import kr_rope

    L, row, last = kq.lib(), 512, 19 * 512
    rope = kr_rope(0x700000, 0x701000, 10, 64, 0, 0)
    bad = [dict(qo=Q + row), dict(qo=Q - row), dict(qo=Q + 16), dict(qo=Q + last + 496), dict(qo=Q - last - 496), dict(qo=K), dict(qo=K - last - 496),
           dict(qo=K + 19 * 256 + 240), dict(qo=V + 256), dict(qo=0x500000 - last - 496), dict(qo=0x500100), dict(qo=0x600000), dict(qo=0x601000),
           dict(qo=0x602000), dict(qo=0x700000, rope=rope), dict(qo=0x701000 - last - 496, rope=rope), dict(qo=0x1000000 + 0x9FF0), dict(qo=0x2000000 - 16),
           dict(k=0x1000000), dict(v=0x1009FF0), dict(k=0x2000000), dict(q=0x2009FF0), dict(layer=1, v=0x100A000), dict(layer=1, q=0x2013FF0),
           dict(norm=kr_head_norm(0x1000000, 0x500100, 1e-6)), dict(norm=kr_head_norm(0x500000, 0x2000000, 1e-6)), dict(table=0x1000000),
           dict(lengths=0x2009FF8), dict(starts=0x1000000 - 4), dict(rope=kr_rope(0x1000000, 0x701000, 10, 64, 0, 0)),
           dict(rope=kr_rope(0x700000, 0x2000000, 10, 64, 0, 0)),
           dict(q=Q, qo=Q + 3 * 512, qs=768),  # rows with gaps: a head of the next row
           dict(q=Q, qo=Q + 256, qs=768), dict(k=Q + 512, kvs=384, qo=Q, q=QO, qs=320)]  # other strides
    for change in bad:
        assert _append(L, **change) == kq.KR_E_INVALID, change
        assert b"overlap" in L.kr_last_error(), change


def test_reads_and_attention_refuse_what_they_write_and_read(kq):
    L = kq.lib()
    cache, step = ctypes.byref(_cache(k=0x1000000, v=0x2000000)), _step(lengths=0x601000, table=0x602000)
    out, lse, ws, q, each = 0x100000, 0x200000, 0x300000, 0x10000000, 2 * 4 * 64 * 2
    for name, at in (("lengths", 0x601000), ("table", 0x602000), ("starts", 0x600000), ("cache k", 0x1000000), ("cache v", 0x2000000)):
        step.starts = 0x600000
        for change in (dict(out=at), dict(out=at - each + 16), dict(lse=at), dict(lse=at - 28), dict(ws=at)):
            a = dict(dict(out=out, lse=lse, ws=ws), **change)
            rc = L.kr_paged_attention(cache, 0, ctypes.byref(step), q, 256, 4, 2, None, 0, 0.125, a["out"], a["lse"], a["ws"], 1 << 30, None)
            assert rc == kq.KR_E_INVALID and b"overlap" in L.kr_last_error(), (name, change)
            assert name.encode() in L.kr_last_error() or "ws" in change  # (so large a workspace may meet several)
    size = 2 * 10 * 2 * 64 * 4
    for k, v in ((0x1000000, 0x100000), (0x100000, 0x2009FF0), (0x601000, 0x100000), (0x100000, 0x602000 - size + 16), (0x700000 - 16, 0x100000),
                 (0x100000, 0x100000 + size - 16)):
        assert L.kr_paged_read(cache, 0, ctypes.byref(step), 0x700000, 10, k, v, 1, None) == kq.KR_E_INVALID, (hex(k), hex(v))
        assert b"overlap" in L.kr_last_error()


def test_commit_refuses_outputs_in_the_pool(kq):
    L, cache, step = kq.lib(), _cache(k=0x1000000, v=0x2000000), _step(lengths=0x601000, table=0x602000)
    for name in range(4):
        for at in (0x1000000, 0x1013FFC, 0x2000000 + 0xA000):  # of the first and of the second layer
            outs = [0x100000, 0x200000, 0x300000, 0x400000]
            outs[name] = at
            assert L.kr_paged_commit(ctypes.byref(cache), ctypes.byref(step), 0x500000, 0x501000, 0x502000, 2, 4, *outs, None) == kq.KR_E_INVALID
            assert b"cache" in L.kr_last_error()
