"""GPU: what the decoder over the paged cache keeps through refused calls, ended sequences and replays past their pages; against steps,
and against the restatement of test_gpu_paged_decode under its bar."""
import numpy as np
import pytest
import torch

from _util import assert_rms_close
from test_gpu_paged_decode import BAR, BATCH, forward_ref, make, stepped  # noqa: F401  (make: the fixture)

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _state(m):
    return [t.clone() for t in (m.lengths, m.positions, m.tokens, m.logits)] + [list(m._used)]


def _same(a, b):
    return all(torch.equal(x, y) if torch.is_tensor(x) else x == y for x, y in zip(a, b))


def _captured(m):
    """A captured step of m, not yet replayed."""
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            m.step()
    torch.cuda.current_stream().wait_stream(side)
    return g


# ---- refused and failed calls

def test_a_refused_verify_changes_nothing(make):
    m = make()
    m.step()
    before, table = _state(m), m.table.clone()
    ids, up = _i32([1, 2, 3]), _i32([-1, 0, -1])
    wide = torch.zeros(3, 2, dtype=I32, device="cuda")
    for tokens, parents, match in ((ids, up.long(), "parents must be torch.int32"), (ids.long(), up, "tokens must be torch.int32"),
                                   (ids, wide[:, 0], "contiguous"), (wide[:, 0], up, "contiguous"), (ids.cpu(), up, "GPU"), (ids, up.cpu(), "GPU"),
                                   (ids[None], up[None], "tokens must be")):
        with pytest.raises(ValueError, match=match):
            m.verify(tokens, parents, [2, 1, 0])
        assert _same(_state(m), before) and torch.equal(m.table, table)
    stepped(m)


def test_a_tree_of_more_nodes_than_a_plan_takes(make):
    m = make(max_ctx=6000)
    before, table = _state(m), m.table.clone()
    nodes = 4097
    with pytest.raises(ValueError, match="4096"):
        m.verify(torch.zeros(nodes, dtype=I32, device="cuda"), torch.arange(-1, nodes - 1, dtype=I32, device="cuda"), [nodes, 0, 0])
    assert _same(_state(m), before) and torch.equal(m.table, table)
    stepped(m)


@pytest.mark.parametrize("late", [False, True])
def test_a_pass_that_fails_changes_nothing(make, monkeypatch, late):
    """An error in the middle of a pass (its first call, or the head's logits): the sequences are as they were."""
    from kriya_q4 import qwen_paged

    m, plain = make(), make()
    m.step()
    plain.step()
    before = _state(m)
    with monkeypatch.context() as patch:
        def fails(*a, **kw):
            raise RuntimeError("out of memory")
        patch.setattr(qwen_paged, "argmax" if late else "embedding", fails)
        for call in (lambda: m.prefill(_i32([1, 2, 3]), [2, 0, 1]), lambda: m.verify(_i32([1, 2, 3]), _i32([-1, 0, -1]), [2, 0, 1])):
            with pytest.raises(RuntimeError, match="out of memory"):
                call()
            assert _same(_state(m)[:3] + [m._used], before[:3] + [before[4]])
    assert torch.equal(m.step(), plain.step()) and torch.equal(m.logits, plain.logits)


def test_verify_of_the_decoders_own_tokens(make):
    """Trees of node 0 alone are a step: `tokens` themselves may be given."""
    m, plain = make(), make()
    path, kept = m.verify(m.tokens, torch.full((BATCH,), -1, dtype=I32, device="cuda"), [1] * BATCH)
    plain.step()
    assert kept.tolist() == [1] * BATCH and path.tolist() == [[0]] * BATCH
    assert m.lengths.tolist() == [41] * BATCH == m.positions.tolist()
    assert torch.equal(m.tokens, plain.tokens)
    stepped(m)


def test_a_prompt_of_the_decoders_own_tokens(make):
    m, plain = make(), make()
    m.prefill(m.tokens, [1] * BATCH)
    plain.step()
    assert torch.equal(m.tokens, plain.tokens) and m.lengths.tolist() == [41] * BATCH
    stepped(m)


def test_prompts_of_other_types_are_refused(make):
    m = make()
    before = _state(m)
    ids = torch.arange(6, device="cuda")
    for tokens, match in ((ids, "torch.int32"), (ids.to(torch.int16), "torch.int32"), (ids.float(), "torch.int32"),
                          (ids.to(I32)[::2].repeat(2)[::2], "contiguous"), (ids.to(I32).cpu(), "GPU")):
        with pytest.raises(ValueError, match=match):
            m.prefill(tokens, [tokens.numel(), 0, 0])
        assert _same(_state(m), before)
    stepped(m)


# ---- sequences that have ended

def _rows(m, tokens, live, lengths, positions):
    counts = [1 if b in live else 0 for b in range(BATCH)]
    return forward_ref(m, tokens[live], counts, lengths, positions[live])


def test_an_ended_sequence_takes_no_part_in_steps(make):
    """Eager: it takes no page and grows no context; a prompt in its place starts from nothing."""
    m = make()
    m.release(1)
    free = len(m._free)
    for i in range(2):
        tokens, positions = m.tokens.cpu().numpy().copy(), m.positions.cpu().clone()
        m.step()
        assert m.lengths.tolist() == [41 + i, 0, 41 + i] == m.positions.tolist()
        want = _rows(m, tokens, [0, 2], [41 + i, 0, 41 + i], positions)
        assert_rms_close(m.logits.cpu().numpy()[[0, 2]], want, rel=BAR, what="the others")
    assert m.table[1].tolist() == [-1] * 8 and len(m._free) == free and torch.isfinite(m.logits).all()
    ids = torch.randint(0, 512, (20,), dtype=I32, generator=torch.Generator().manual_seed(6))
    m.prefill(ids.cuda(), [0, 20, 0])
    assert m.lengths.tolist() == [42, 20, 42] == m.positions.tolist()
    want = forward_ref(m, ids.numpy(), [0, 20, 0], [42, 20, 42], torch.arange(20, dtype=I32))
    assert_rms_close(m.logits.cpu().numpy()[[1]], want[[19]], rel=BAR, what="prompt after the release")
    stepped(m)
    assert m.lengths.tolist() == [43, 21, 43]


def test_ended_sequences_need_no_pages(make):
    """A pool that is full but for one sequence's page goes on once the others have ended."""
    m = make(pages=9)  # three pages each, of which 8 slots are left
    for _ in range(8):
        m.step()
    with pytest.raises(ValueError, match="release"):
        m.step()
    m.release(0)
    m.release(2)
    for _ in range(20):
        m.step()
    m.reserve(10)
    assert m.lengths.tolist() == [0, 68, 0] and [len(p) for p in m._pages] == [0, 5, 0]


def test_captured_steps_after_a_release(make):
    """Replays pass an ended sequence over, and take it along once a prompt has filled its place: all as eager steps do."""
    m, eager = make(), make()
    ids = torch.randint(0, 512, (20,), dtype=I32, generator=torch.Generator().manual_seed(7)).cuda()
    m.step(), eager.step()
    m.reserve(40)
    g = _captured(m)

    def both(n):
        for _ in range(n):
            g.replay()
            eager.step()
            torch.cuda.synchronize()
            torch.ones(1000, device="cuda").sum().item()
            assert torch.equal(m.lengths, eager.lengths) and torch.equal(m.positions, eager.positions)
            live = m.lengths > 0
            assert torch.equal(m.logits[live], eager.logits[live]) and torch.equal(m.tokens[live], eager.tokens[live])
    both(2)
    m.release(1), eager.release(1)
    both(3)
    assert m.lengths.tolist() == [46, 0, 46] and m.table[1].max() < 0
    for x in (m, eager):
        x.step()
        x.prefill(ids, [0, 20, 0])
    m.reserve(20)
    both(12)
    assert m.lengths.tolist() == [59, 32, 59]
    stepped(m)


def test_a_sequence_past_its_pages_is_released_and_the_others_go_on(make):
    m = make()
    m.prefill(torch.arange(5, dtype=I32).cuda(), [5, 0, 0])
    m.step()  # 46, 41, 41 tokens in three pages each
    g = _captured(m)
    for _ in range(4):
        g.replay()
    for call in (m.step, lambda: m.reserve(1), lambda: m.prefill(m.tokens[:1], [0, 1, 0])):
        with pytest.raises(RuntimeError, match="reserve before"):
            call()
    m.release(0)
    assert m.lengths.tolist() == [0, 45, 45] and m.table[0].max() < 0
    tokens, positions = m.tokens.cpu().numpy().copy(), m.positions.cpu().clone()
    m.step()
    want = _rows(m, tokens, [1, 2], [0, 46, 46], positions)
    assert_rms_close(m.logits.cpu().numpy()[[1, 2]], want, rel=BAR, what="the others")
    m.prefill(torch.arange(9, dtype=I32).cuda(), [9, 0, 0])
    m.reserve(4)
    g.replay()
    assert m.lengths.tolist() == [10, 47, 47]
    stepped(m)
    used = [p for row in m.table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) and sorted(used + m._free) == list(range(m.cache.pages))


def test_all_sequences_past_their_pages_are_released_one_by_one(make):
    m = make()
    m.step()
    g = _captured(m)
    for _ in range(8):
        g.replay()
    for b in range(BATCH):
        with pytest.raises(RuntimeError, match="reserve before"):
            m.reserve(1)
        m.release(b)
    assert m.lengths.tolist() == [0] * BATCH and len(m._free) == m.cache.pages
    m.prefill(torch.arange(6, dtype=I32).cuda(), [1, 2, 3])
    stepped(m)


def test_a_tree_starts_an_ended_sequence_again(make):
    m = make()
    m.release(2)
    path, kept = m.verify(_i32([7, 9]), _i32([-1, -1]), [0, 0, 2])
    assert kept.tolist() == [0, 0, 1] and m.lengths.tolist() == [40, 40, 1]
    stepped(m)


def test_sequences_that_are_none(make):
    m = make()
    before = _state(m)
    for b in (-1, BATCH, BATCH + 4):
        with pytest.raises(ValueError, match="sequence"):
            m.release(b)
        assert _same(_state(m), before) and len(m._free) == m.cache.pages - 3 * BATCH
    m.release(0)
    m.release(0)  # nothing left to end
    assert len(m._free) == m.cache.pages - 6 and m.lengths.tolist() == [0, 40, 40]
