"""GPU: the decoder over the 8-bit cache, the calls run together as a program runs them: ragged prompts, decoding, captured
steps, eviction; against a layer-by-layer restatement on the CPU over the values that the device's caches stand for.

Bar: max |gpu - cpu| <= 3e-2 * RMS(cpu) for logits, as for the bf16 decoder at small sizes.  Device and restatement round to
bf16 at the same points, but probabilities are fp16 on the device (2^-12 of a value off), so values near a tie round the
other way and by the second layer any may: an ulp of bf16 is 2^-8 to 2^-7 of its value, on average 0.7 * 2^-7 = 5.4e-3.  A logit is a sum
of 256 products, so its error from one such rounding of every h is 5.4e-3 of the logits' RMS, from two (h, and its norm x) 7.6e-3, and
the largest of 1536 logits is 3.5 to 4 times that: 3e-2.  (The bf16 decoder at these sizes: 9e-6 to 4.6e-2 over eight seeds.)
Two device paths that each keep it differ by at most twice that."""
import itertools

import numpy as np
import pytest
import torch

import _kv8_ref as ref
import oracle as O
from _decode_ref import bf, f32, planar
from _util import assert_rms_close, rms

pytestmark = pytest.mark.gpu
BATCH, CTX = 3, 40
BAR = 3e-2


@pytest.fixture(scope="module")
def make(kq):
    from kriya_q4.qwen_decode import QwenConfig
    from kriya_q4.qwen_kv8 import QwenKv8Decoder

    cfg = QwenConfig(hidden=256, inter=384, layers=2, vocab=512, q_heads=4, kv_heads=2, head_dim=64, rope_theta=1e4)

    def f(**kw):
        m = QwenKv8Decoder(cfg, **dict(dict(batch=BATCH, ctx=CTX, seed=11, max_ctx=128), **kw))
        for L in m.layers:  # keep each layer's output near its input's size
            for w in (L.q, L.k, L.v, L.o, L.gate, L.up, L.down):
                w.scales.view(torch.bfloat16).mul_(0.25)
                w.biases.view(torch.bfloat16).mul_(0.25)
        return m
    return f


def forward_ref(m, tokens, spans, positions):
    """Logits of the tokens ([n], sequence after sequence, spans [(first row, count, length)], rope positions) after a device
    pass: everything again on the CPU, with attention over what the device's caches now hold."""
    c = m.cfg
    E, cs = planar(m.embed), m.cos_sin.cpu()
    h = bf(O.dequant_planar(E)[tokens])
    starts = torch.tensor([s[0] for s in spans] + [len(tokens)])
    lengths = torch.tensor([s[2] for s in spans])

    def norm(v, w):
        return bf(v / np.sqrt((v.astype(np.float64) ** 2).mean(axis=1, keepdims=True) + c.eps) * f32(w))

    def mm(W, v):
        return O.q4_matmul(planar(W), O.f32_to_bf16(v))
    for L in m.layers:
        x = norm(h, L.ln1)
        q, k, v = (bf(mm(W, x) + f32(b)).reshape(len(tokens), -1, c.head_dim) for W, b in ((L.q, L.bq), (L.k, L.bk), (L.v, L.bv)))
        q, k = (bf(ref.rope64(torch.from_numpy(t), cs, positions, 0).numpy()) for t in (q, k))
        kc, vc = ref.read(L.cache, m.lengths.max())
        m_code = 127.0 if L.cache.format == 0 else 448.0
        for (b, (t0, n, total)), (cache, new, scale) in itertools.product(enumerate(spans), ((kc, k, L.cache.k_scale), (vc, v, L.cache.v_scale))):
            for i in range(n):  # the new rows: half a code (e4m3: of the largest binade) and the matmul's bar
                p = total - n + i
                step = scale[b, :, p // 32].cpu().double().numpy()[:, None] * (0.5 if m_code == 127.0 else 16.0)
                off = np.abs(cache[b, :, p].numpy() - new[t0 + i])
                assert (off <= step + 2e-2 * rms(new) + 2.0 ** -8 * np.abs(new[t0 + i])).all()
        a = ref.attention(torch.from_numpy(q), kc, vc, starts, lengths, c.head_dim ** -0.5, kc.shape[2])[0]
        h = bf(h + mm(L.o, bf(a.numpy().reshape(len(tokens), -1))))
        x = norm(h, L.ln2)
        g, u = mm(L.gate, x), mm(L.up, x)
        h = bf(h + mm(L.down, bf(g / (1.0 + np.exp(-g)) * u)))
    return O.q4_matmul(E, O.f32_to_bf16(norm(h, m.ln_f)))


@pytest.mark.parametrize("format", [0, 1])
def test_steps(make, format):
    m = make(format=format)
    for _ in range(2):
        tokens, pos, n = m.tokens.cpu().numpy().copy(), m.positions.cpu().clone(), m.lengths.cpu() + 1
        nxt = m.step().cpu().numpy()
        assert torch.equal(m.lengths.cpu(), n) and torch.equal(m.positions.cpu(), pos + 1)
        want = forward_ref(m, tokens, [(b, 1, int(n[b])) for b in range(BATCH)], pos)
        assert_rms_close(m.logits.cpu().numpy(), want, rel=BAR, what="step")
        assert np.array_equal(nxt, m.logits.cpu().numpy().argmax(axis=1))


def test_ragged_prompts_then_steps(make):
    """Prompts of 37, 0 and 1 tokens on top of what the caches hold, as one batch; the same tokens one by one; then a step."""
    counts = [37, 0, 1]
    ids = torch.randint(0, 512, (38,), dtype=torch.int32, generator=torch.Generator().manual_seed(5))
    m, one = make(), make()
    before = m.logits.fill_(7.0).clone()
    m.prefill(ids.cuda(), counts)
    assert m.lengths.tolist() == [77, 40, 41] and m.positions.tolist() == [77, 40, 41]
    pos = torch.cat([torch.arange(40, 77), torch.tensor([40])]).to(torch.int32)
    want = forward_ref(m, ids.numpy(), [(0, 37, 77), (37, 0, 40), (37, 1, 41)], pos)
    got = m.logits.cpu().numpy()
    assert_rms_close(got[[0, 2]], want[[36, 37]], rel=BAR, what="prompt")
    assert torch.equal(m.logits[1], before[1])
    assert m.tokens[0] == got[0].argmax() and m.tokens[2] == got[2].argmax()
    # one by one: sequence 0's tokens through prompts of one
    for i in range(37):
        one.prefill(ids[[i] if i else [0, 37]].cuda(), [1, 0, 0 if i else 1])
    two = one.logits.cpu().numpy()
    assert np.abs(two[[0, 2]] - got[[0, 2]]).max() <= 2 * BAR * rms(got[[0, 2]])
    tokens, n = m.tokens.cpu().numpy().copy(), m.lengths.cpu() + 1
    p = m.positions.cpu().clone()
    m.step()
    want = forward_ref(m, tokens, [(b, 1, int(n[b])) for b in range(BATCH)], p)
    assert_rms_close(m.logits.cpu().numpy(), want, rel=BAR, what="step after the prompt")


def test_captured_steps(make):
    """Five replays of a captured step, with eager work and synchronizations between, give five eager steps' bits."""
    eager, m = make(track_weights=True), make(track_weights=True)
    want = []
    for _ in range(6):
        eager.step()
        want.append((eager.logits.clone(), eager.tokens.clone()))
    m.step()  # loads the code
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            m.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(m.logits, want[0][0]) and m.lengths.tolist() == [41] * BATCH
    for logits, tokens in want[1:]:
        g.replay()
        torch.cuda.synchronize()
        torch.ones(1000, device="cuda").sum().item()
        assert torch.equal(m.logits, logits) and torch.equal(m.tokens, tokens)
    for a, b in zip(eager.layers, m.layers):
        assert torch.equal(a.weight[..., :46], b.weight[..., :46])
        assert all(torch.equal(x, y) for x, y in zip(ref.read(a.cache, 46), ref.read(b.cache, 46)))


def test_evict_and_go_on(make):
    """Steps that track the weights, an eviction of every layer, further steps and a prompt over what is left."""
    m = make(track_weights=True, max_ctx=64, max_positions=200)
    for _ in range(9):
        m.step()
    sums = [L.weight[:, :, :49].sum(-1) for L in m.layers]
    for s in sums:  # each of 9 tokens adds 1 for each of the group's two heads
        assert (s - 18.0).abs().max() <= 1e-3
    old = [(ref.read(L.cache, 49), L.weight.cpu()) for L in m.layers]
    m.evict(30, sink=2, recent=10)
    assert m.lengths.tolist() == [30] * BATCH and m.positions.tolist() == [49] * BATCH
    for L, ((k, v), w) in zip(m.layers, old):
        nk, nv = ref.read(L.cache, 30)
        for b in range(BATCH):
            for h in range(2):
                slots = ref.kept_slots(w[b, h], 49, 30, 2, 10)
                assert torch.equal(L.weight[b, h, :30].cpu(), w[b, h, slots])
                for new, was, scale in ((nk, k, L.cache.k_scale), (nv, v, L.cache.v_scale)):  # coded again: half a code, and of the last block the raw rows' half code before
                    off = (new[b, h] - was[b, h, slots]).abs().max()
                    assert off <= 0.51 * float(scale[b, h, 0]) + 0.51 * float(was[b, h].abs().max()) / 127 + 2.0 ** -8 * float(was[b, h].abs().max())
    for _ in range(2):
        tokens, p, n = m.tokens.cpu().numpy().copy(), m.positions.cpu().clone(), m.lengths.cpu() + 1
        m.step()
        want = forward_ref(m, tokens, [(b, 1, int(n[b])) for b in range(BATCH)], p)
        assert_rms_close(m.logits.cpu().numpy(), want, rel=BAR, what="step after the eviction")
    ids = torch.arange(20, dtype=torch.int32)
    m.prefill(ids.cuda(), [0, 20, 0])
    want = forward_ref(m, ids.numpy(), [(0, 0, 32), (0, 20, 52), (20, 0, 32)], torch.arange(51, 71, dtype=torch.int32))
    assert_rms_close(m.logits.cpu().numpy()[[1]], want[[19]], rel=BAR, what="prompt after the eviction")


def test_sequences_grow_for_themselves_and_positions_end(make):
    """Prompts of one sequence each that only fit one by one are taken; positions past the rotary table are refused, before
    anything has changed."""
    m = make(max_ctx=64, max_positions=66, track_weights=True)
    ids = torch.zeros(24, dtype=torch.int32, device="cuda")
    for b in range(BATCH):
        m.prefill(ids, [24 * (i == b) for i in range(BATCH)])
    assert m.lengths.tolist() == [64] * BATCH
    with pytest.raises(ValueError, match="evict first"):
        m.step()
    m.evict(20, sink=2, recent=10)
    m.step()
    m.step()
    with pytest.raises(ValueError, match="max_positions"):
        m.step()
    with pytest.raises(ValueError, match="max_positions"):
        m.prefill(ids[:1], [0, 1, 0])
    assert m.lengths.tolist() == [22] * BATCH and m.positions.tolist() == [66] * BATCH


def test_refusals(make):
    m = make(max_ctx=42)
    m.step()
    m.step()
    with pytest.raises(ValueError, match="evict first"):
        m.step()
    with pytest.raises(ValueError, match="track_weights"):
        m.evict(10)
    with pytest.raises(ValueError, match="counts"):
        m.prefill(torch.zeros(3, dtype=torch.int32, device="cuda"), [1, 1])
    with pytest.raises(ValueError, match="max_ctx"):
        make(max_ctx=39)
