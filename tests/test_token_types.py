"""Token ids of another type than the kernels read are refused: on the CPU the lookup itself, on the GPU the 8-bit cache's decoder,
whose sequences stay as they were (the paged cache's decoder: test_gpu_paged_decode_state.py)."""
import types

import pytest
import torch

OTHERS = [torch.int64, torch.int16, torch.uint8, torch.float32, torch.bool]


@pytest.mark.parametrize("dtype", OTHERS)
def test_embedding_refuses_other_types(dtype):
    import kriya_q4

    table = types.SimpleNamespace(k=64, desc=None)  # nothing of it is reached
    with pytest.raises(ValueError, match="torch.int32"):
        kriya_q4.embedding(table, torch.zeros(4).to(dtype))
    with pytest.raises(ValueError, match="contiguous"):
        kriya_q4.embedding(table, torch.zeros(8, dtype=torch.int32)[::2])
    with pytest.raises(ValueError, match="GPU"):  # the type is right
        kriya_q4.embedding(table, torch.zeros(4, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", OTHERS)
def test_the_8_bit_caches_decoder_refuses_them(kq, dtype):
    from kriya_q4.qwen_decode import QwenConfig
    from kriya_q4.qwen_kv8 import QwenKv8Decoder

    m = QwenKv8Decoder(QwenConfig(hidden=256, inter=384, layers=1, vocab=512, q_heads=4, kv_heads=2, head_dim=64), batch=2, ctx=8, max_ctx=32)
    ids = torch.tensor([3, 1, 4], device="cuda")
    with pytest.raises(ValueError, match="torch.int32"):
        m.prefill(ids.to(dtype), [2, 1])
    assert m.lengths.tolist() == [8, 8] == m.positions.tolist() and m._used == [8, 8]
    m.prefill(ids.to(torch.int32), [2, 1])
    assert m.lengths.tolist() == [10, 9]
