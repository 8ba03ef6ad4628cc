"""GPU: the decoder over the 8-bit cache after replays of a captured step, which its host never sees: prompts, steps and
evictions go by the lengths and positions on the device."""
import pytest
import torch

from test_gpu_kv8_decode import BATCH, make  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def _captured(m):
    m.step()  # loads the code
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            m.step()
    torch.cuda.current_stream().wait_stream(side)
    return g


def _ids(n):
    return torch.arange(n, dtype=torch.int32, device="cuda") % 512


def test_a_prompt_after_replays_fits_or_is_refused(make):
    m = make()  # 40 of 128 slots
    g = _captured(m)
    for _ in range(59):
        g.replay()
    assert m.lengths.tolist() == [100] * BATCH
    before = m.logits.clone()
    with pytest.raises(ValueError, match="evict first"):
        m.prefill(_ids(29), [0, 29, 0])
    assert m.lengths.tolist() == [100] * BATCH and torch.equal(m.logits, before)
    m.prefill(_ids(28), [0, 28, 0])
    assert m.lengths.tolist() == [100, 128, 100] and m.positions.tolist() == [100, 128, 100]


def test_an_eager_step_after_replays_fits_or_is_refused(make):
    m = make(max_ctx=64)
    g = _captured(m)
    for _ in range(22):
        g.replay()
    m.step()
    assert m.lengths.tolist() == [64] * BATCH
    with pytest.raises(ValueError, match="evict first"):
        m.step()
    assert m.lengths.tolist() == [64] * BATCH


def test_an_eviction_after_replays_counts_what_is_left(make):
    m = make(track_weights=True, max_positions=240)
    g = _captured(m)
    for _ in range(80):
        g.replay()
    m.evict(60, recent=40)
    assert m.lengths.tolist() == [60] * BATCH
    with pytest.raises(ValueError, match="evict first"):
        m.prefill(_ids(80), [80, 0, 0])
    m.prefill(_ids(68), [68, 0, 0])
    m.prefill(_ids(8), [0, 4, 4])
    assert m.lengths.tolist() == [128, 64, 64] and m.positions.tolist() == [189, 125, 125]


def test_positions_after_replays_end_with_the_table(make):
    m = make(track_weights=True, max_positions=110)
    g = _captured(m)
    for _ in range(64):
        g.replay()
    m.evict(20, sink=2, recent=10)
    with pytest.raises(ValueError, match="max_positions"):
        m.prefill(_ids(6), [0, 0, 6])
    m.prefill(_ids(5), [0, 0, 5])
    m.evict(20, sink=2, recent=10)
    with pytest.raises(ValueError, match="max_positions"):
        m.step()
    assert m.lengths.tolist() == [20] * BATCH and m.positions.tolist() == [105, 105, 110]


def test_prompts_and_evictions_are_refused_inside_a_capture(make):
    m = make(track_weights=True)
    m.step()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            m.step()
            with pytest.raises(RuntimeError, match="capture"):
                m.prefill(m.tokens, [1, 1, 1])
            with pytest.raises(RuntimeError, match="capture"):
                m.evict(30)
    torch.cuda.current_stream().wait_stream(side)
    g.replay()
    assert m.lengths.tolist() == [42] * BATCH
