"""GPU: the buffers that the 8-bit cache's and the rotary calls make for themselves on another stream than the current one."""
import pytest
import torch

from test_gpu_kv8 import _fill, _i32, _rand, _starts, kv8  # noqa: F401  (kv8: the fixture)

pytestmark = pytest.mark.gpu


def _pool(t):
    """The stream whose memory t lies in."""
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= t.data_ptr() < s["address"] + s["total_size"]:
            return s["stream"]


def _setup(kv8):
    g = torch.Generator().manual_seed(41)
    cache = _fill(kv8, g, [3000, 2000], 2, 64, 0, 3000)
    q, lens, starts = _rand(g, 400, 8, 64).cuda(), _i32([3000, 2000]), _starts([300, 100])
    return cache, q, lens, starts, torch.rand(2, 2, 3000, generator=g).cuda()


def _calls(kv8, rope, cache, q, lens, starts, weight, stream):
    """Every call that makes a buffer, and the tensors that came of it."""
    out, lse = kv8.attention(cache, q, lens, starts=starts, stream=stream)
    w = weight.clone()
    if stream is not None:
        raw = stream if isinstance(stream, int) else stream.cuda_stream
        torch.cuda.ExternalStream(raw).wait_stream(torch.cuda.current_stream())
    kv8.accumulate_weight(cache, q, lse, lens, w, starts=starts, stream=stream)
    to, to_weight = kv8.Kv8Cache(2, 2, 64, 1000), torch.zeros(2, 2, 1000, device="cuda")
    if stream is not None:
        torch.cuda.ExternalStream(raw).wait_stream(torch.cuda.current_stream())
    kept, left = kv8.evict(cache, lens, weight, 1000, 4, 100, to, to_weight, stream=stream)
    k, v = kv8.dequant(to, left, 1000, stream=stream)
    table = rope.table(64, 4000, 1e6, stream=stream)
    return (out, lse, kept, left, k, v, table), (w, to_weight)


@pytest.mark.parametrize("raw", [False, True])
def test_buffers_lie_in_the_calls_own_streams_memory(kv8, monkeypatch, raw):
    from kriya_q4 import rope

    data, side, spaces = _setup(kv8), torch.cuda.Stream(), []
    want = [t.clone() for ts in _calls(kv8, rope, *data, None) for t in ts]
    for name in ("attention_workspace", "weight_workspace"):
        make = getattr(kv8, name)
        monkeypatch.setattr(kv8, name, lambda *a, make=make: spaces.append(make(*a)) or spaces[-1])
    torch.cuda.synchronize()
    made, given = _calls(kv8, rope, *data, side.cuda_stream if raw else side)
    assert [_pool(t) for t in made] == [side.cuda_stream] * len(made)
    assert len(spaces) == 2 and [_pool(t) for t in spaces] == [side.cuda_stream] * 2
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(made + given, want))
    # the current stream, given by name: nothing changes hands
    made, given = _calls(kv8, rope, *data, torch.cuda.current_stream())
    assert side.cuda_stream not in [_pool(t) for t in made]
    assert all(torch.equal(a, b) for a, b in zip(made + given, want))


def test_buffers_do_not_meet_work_that_is_pending_on_the_current_stream(kv8):
    """Memory that the current stream has given back but still writes is not what a call on another stream gets; and a result that
    is dropped early is not reused while the call still needs it (evict reads `kept` in its second kernel)."""
    cache, q, lens, starts, weight = _setup(kv8)
    want = kv8.attention(cache, q, lens, starts=starts)
    to, to_weight = kv8.Kv8Cache(2, 2, 64, 1000), torch.zeros(2, 2, 1000, device="cuda")
    kv8.evict(cache, lens, weight, 1000, 4, 100, to, to_weight)
    got, got_weight = kv8.Kv8Cache(2, 2, 64, 1000), torch.zeros(2, 2, 1000, device="cuda")
    for x, y in zip((got.k, got.v, got.k_scale, got.v_scale), (to.k, to.v, to.k_scale, to.v_scale)):
        x.copy_(y)  # (bytes behind the last slot, which no call writes)
        x[:, :, : 1000 // 32].zero_()
    n = kv8.attention_workspace(cache, 8, 400).numel()
    sizes = [n, want[0].numel() * 2, want[1].numel() * 4, 2 * 2 * 1000 * 4]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(20_000_000)  # about 10 ms
    for x in [torch.empty(s, dtype=torch.uint8, device="cuda") for s in sizes]:
        x.fill_(255)
        del x
    out, lse = kv8.attention(cache, q, lens, starts=starts, stream=side)
    kv8.evict(cache, lens, weight, 1000, 4, 100, got, got_weight, stream=side)
    for s in sizes:
        torch.full((s,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert torch.equal(got_weight, to_weight)
    assert all(torch.equal(x, y) for x, y in zip((got.k, got.v, got.k_scale, got.v_scale), (to.k, to.v, to.k_scale, to.v_scale)))
