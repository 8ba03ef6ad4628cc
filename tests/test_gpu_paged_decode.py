"""GPU: the decoder over the paged cache, its calls run together as a server runs them: ragged prompts, decoding, captured steps,
drafted trees, sequences that end; against a layer-by-layer restatement on the CPU over what the device's pages hold.

Bar: max |gpu - cpu| <= 3e-2 * RMS(cpu) for logits, as for the decoder over the 8-bit cache and for its reasons: both sides round to
bf16 at the same points, and a value near a tie may round the other way; the probabilities, bf16 here in tiles of many rows, are off
by up to 2^-8 of themselves, which moves a result by at most as much as its own rounding does.  Two device paths that each keep it differ by at most twice that."""
import numpy as np
import pytest
import torch

import _kv8_ref
import _paged_ref as ref
import oracle as O
from _decode_ref import bf, f32, planar
from _util import assert_rms_close, rms

pytestmark = pytest.mark.gpu
BATCH, CTX, PAGE = 3, 40, 16
BAR = 3e-2


@pytest.fixture(scope="module")
def make(kq):
    from kriya_q4.qwen_decode import QwenConfig
    from kriya_q4.qwen_paged import QwenPagedDecoder

    cfg = QwenConfig(hidden=256, inter=384, layers=2, vocab=512, q_heads=4, kv_heads=2, head_dim=64, rope_theta=1e4)

    def f(**kw):
        m = QwenPagedDecoder(cfg, **dict(dict(batch=BATCH, ctx=CTX, seed=11, max_ctx=128, page=PAGE), **kw))
        for L in m.layers:  # keep each layer's output near its input's size
            for w in (L.q, L.k, L.v, L.o, L.gate, L.up, L.down):
                w.scales.view(torch.bfloat16).mul_(0.25)
                w.biases.view(torch.bfloat16).mul_(0.25)
        return m
    return f


def pages_of(m, layer):
    """[(k, v)] of every sequence, f64 [kv_heads, slots, head_dim]."""
    out = []
    for row in m.table.tolist():
        pages = [None if p < 0 else p for p in row]
        out.append(tuple(ref.slots_of(x[layer], w, pages, PAGE) for x, w in ((m.cache.k, "k"), (m.cache.v, "v"))))
    return out


def forward_ref(m, tokens, counts, lengths, positions, masks=None):
    """Logits of the tokens ([n], sequence after sequence) after a device pass that brought the sequences to `lengths`: everything
    again on the CPU, with attention over what the device's pages now hold."""
    c = m.cfg
    E, cs = planar(m.embed), m.cos_sin.cpu()
    h = bf(O.dequant_planar(E)[tokens])

    def norm(v, w):
        return bf(v / np.sqrt((v.astype(np.float64) ** 2).mean(axis=1, keepdims=True) + c.eps) * f32(w))

    def mm(W, v):
        return O.q4_matmul(planar(W), O.f32_to_bf16(v))
    for i, L in enumerate(m.layers):
        x = norm(h, L.ln1)
        q, k, v = (bf(mm(W, x) + f32(b)).reshape(len(tokens), -1, c.head_dim) for W, b in ((L.q, L.bq), (L.k, L.bk), (L.v, L.bv)))
        q, k = (bf(_kv8_ref.rope64(torch.from_numpy(t), cs, positions, 0).numpy()) for t in (q, k))
        a, t0 = np.zeros_like(q), 0
        for b, ((kc, vc), n, total) in enumerate(zip(pages_of(m, i), counts, lengths)):
            for cache, new in ((kc, k), (vc, v)):  # the new rows: the matmul's bar and a rounding
                off = np.abs(cache[:, total - n: total].transpose(0, 1).numpy() - new[t0: t0 + n])
                assert n == 0 or (off <= 2e-2 * rms(new) + 2.0 ** -8 * np.abs(new[t0: t0 + n])).all()
            seen = ref.sees(n, total, kc.shape[1], None if masks is None else masks[b])
            a[t0: t0 + n] = ref.attention(torch.from_numpy(q[t0: t0 + n]).double(), kc, vc, seen, c.head_dim ** -0.5)[0].numpy()
            t0 += n
        h = bf(h + mm(L.o, bf(a.reshape(len(tokens), -1))))
        x = norm(h, L.ln2)
        g, u = mm(L.gate, x), mm(L.up, x)
        h = bf(h + mm(L.down, bf(g / (1.0 + np.exp(-g)) * u)))
    return O.q4_matmul(E, O.f32_to_bf16(norm(h, m.ln_f)))


def stepped(m):
    """A step, held against the restatement."""
    tokens, pos, n = m.tokens.cpu().numpy().copy(), m.positions.cpu().clone(), m.lengths.cpu() + 1
    nxt = m.step().cpu().numpy()
    assert torch.equal(m.lengths.cpu(), n) and torch.equal(m.positions.cpu(), pos + 1)
    assert_rms_close(m.logits.cpu().numpy(), forward_ref(m, tokens, [1] * m.batch, n.tolist(), pos), rel=BAR, what="step")
    assert np.array_equal(nxt, m.logits.cpu().numpy().argmax(axis=1))


def test_prompts_and_steps(make):
    """Prompts of 37, 0 and 1 tokens on top of what the pages hold, as one batch; then steps."""
    m = make()
    stepped(m)
    ids = torch.randint(0, 512, (38,), dtype=torch.int32, generator=torch.Generator().manual_seed(5))
    before = m.logits.fill_(7.0).clone()
    m.prefill(ids.cuda(), [37, 0, 1])
    assert m.lengths.tolist() == [78, 41, 42] and m.positions.tolist() == [78, 41, 42]
    pos = torch.cat([torch.arange(41, 78), torch.tensor([41])]).to(torch.int32)
    want = forward_ref(m, ids.numpy(), [37, 0, 1], [78, 41, 42], pos)
    got = m.logits.cpu().numpy()
    assert_rms_close(got[[0, 2]], want[[36, 37]], rel=BAR, what="prompt")
    assert torch.equal(m.logits[1], before[1])
    assert m.tokens[0] == got[0].argmax() and m.tokens[2] == got[2].argmax()
    for _ in range(2):
        stepped(m)


def test_drafted_trees(make):
    """Trees around the model's own greedy tokens: the pass's logits are the restatement's, the path kept is theirs, and steps go on
    behind it as behind the same tokens of decoding."""
    plain, m = make(), make()
    greedy = [plain.tokens.tolist()]
    for _ in range(4):
        plain.step()
        greedy.append(plain.tokens.tolist())
    other = lambda x: (x + 1) % 512  # noqa: E731
    g = [[row[b] for row in greedy] for b in range(BATCH)]
    # sequence 0: a chain of three choices behind node 0, with wrong siblings before and after; 1: nothing; 2: node 0 and wrong ones
    tokens = [g[0][0], other(g[0][1]), g[0][1], g[0][2], other(g[0][3]), g[0][3], g[0][4]] + [g[2][0], other(g[2][1]), g[2][2]]
    parents = [-1, 0, 0, 2, 3, 3, 1] + [-1, 0, 1]
    counts, start = [7, 0, 3], m.lengths.tolist()
    before = m.tokens.tolist()
    path, kept = m.verify(torch.tensor(tokens, dtype=torch.int32).cuda(), torch.tensor(parents, dtype=torch.int32).cuda(), counts)
    assert kept.tolist() == [4, 0, 1] and path[0, :4].tolist() == [0, 2, 3, 5] and path[2, 0] == 0
    assert m.lengths.tolist() == [start[0] + 4, start[1], start[2] + 1] == m.positions.tolist()
    assert m.tokens.tolist() == [g[0][4], before[1], g[2][1]]
    # the rows kept are those of the steps: as prompts of those tokens over the same contexts (causal) on the CPU
    want = forward_ref(m, np.array([g[0][0], g[0][1], g[0][2], g[0][3], g[2][0]]), [4, 0, 1], m.lengths.tolist(),
                       torch.tensor([40, 41, 42, 43, 40], dtype=torch.int32))
    assert_rms_close(m.logits.cpu().numpy()[[0, 2]], want[[3, 4]], rel=BAR, what="tree")
    assert np.abs(m.logits[0].cpu().numpy() - plain.logits[0].cpu().numpy()).max() <= 2 * BAR * rms(want)
    for _ in range(2):
        stepped(m)


def test_captured_steps(make):
    """Replays of a captured step, with eager work and synchronizations between, give eager steps' bits, across pages' ends."""
    eager, m = make(), make()
    want = []
    for _ in range(12):
        eager.step()
        want.append((eager.logits.clone(), eager.tokens.clone()))
    m.step()  # loads the code
    m.reserve(10)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            m.step()
            for call in (lambda: m.prefill(m.tokens, [1] * BATCH), lambda: m.verify(m.tokens, m.tokens, [1] * BATCH),
                         lambda: m.release(0), lambda: m.reserve(1)):
                with pytest.raises(RuntimeError, match="capture"):
                    call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(m.logits, want[0][0]) and m.lengths.tolist() == [41] * BATCH
    for logits, tokens in want[1:11]:
        g.replay()
        torch.cuda.synchronize()
        torch.ones(1000, device="cuda").sum().item()
        assert torch.equal(m.logits, logits) and torch.equal(m.tokens, tokens)
    m.step()  # goes by the lengths on the device
    assert torch.equal(m.logits, want[11][0]) and m.lengths.tolist() == [52] * BATCH
    m.reserve(1)
    g.replay()
    m.step()  # and so after a reserve
    assert m.lengths.tolist() == [54] * BATCH and m.table[:, 3].min() >= 0
    for _ in range(11):  # past the four pages
        g.replay()
    for call in (m.step, lambda: m.reserve(1), lambda: m.prefill(m.tokens, [1] * BATCH)):
        with pytest.raises(RuntimeError, match="reserve before"):
            call()


def test_sequences_end_and_make_room(make):
    """A pool that all sequences' whole contexts would not fit: refused before anything has changed, until one ends; its pages serve
    another, and a new prompt starts from nothing."""
    m = make(pages=11)  # three sequences of three pages each and two
    ids = torch.arange(60, dtype=torch.int32)
    m.prefill(ids[:30].cuda(), [30, 0, 0])  # two more pages
    with pytest.raises(ValueError, match="release"):
        m.prefill(ids[:10].cuda(), [0, 10, 0])
    assert m.lengths.tolist() == [70, 40, 40]
    m.release(0)
    assert m.lengths.tolist() == [0, 40, 40] and m.table[0].tolist() == [-1] * 8
    m.prefill(ids[:50].cuda(), [10, 40, 0])
    want = forward_ref(m, ids[:50].numpy(), [10, 40, 0], [10, 80, 40], torch.cat([torch.arange(10), torch.arange(40, 80)]).to(torch.int32))
    assert_rms_close(m.logits.cpu().numpy()[[0, 1]], want[[9, 49]], rel=BAR, what="prompt after the release")
    used = [p for row in m.table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 1 + 5 + 3
    stepped(m)


def test_refusals(make):
    m = make(max_ctx=41)
    m.step()
    with pytest.raises(ValueError, match="max_ctx"):
        m.step()
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="counts"):
        m.prefill(ids, [1, 1])
    with pytest.raises(ValueError, match="counts"):
        m.verify(ids, ids, [4, -1, 0])
    with pytest.raises(ValueError, match="parents"):
        m.verify(ids, ids[:2], [1, 1, 1])
    with pytest.raises(ValueError, match="max_ctx"):
        m.verify(ids, ids, [1, 1, 1])
    assert m.lengths.tolist() == [41] * BATCH
    path, kept = m.verify(ids[:0], ids[:0], [0, 0, 0])
    assert kept.tolist() == [0] * BATCH
    with pytest.raises(ValueError, match="max_ctx"):
        make(max_ctx=39)
