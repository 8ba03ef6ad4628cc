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
