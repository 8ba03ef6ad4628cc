"""The Qwen2.5-shaped decoder of kriya_q4.qwen_decode over an 8-bit key/value cache: prompts as ragged batches, decoding at
growing positions, rotary tables stretched for long contexts, and eviction by accumulated attention weight.

A layer is that of qwen_decode, with its attention block in these calls:

    q, k, v = rmsnorm(h, ln1) Wq^T + bq, ...           encode_fused_qkv (encoder.rs:2539-2619)
    rope(q, k) at the positions; k, v into the cache   kv8.append, one launch
    a, lse = attention(q, K, V)                        kv8.attention, causal at the cache's end
    weight += e^(scores - lse) by slot                 kv8.accumulate_weight (track_weights)
    h += a Wo^T                                        encode_q4_linear_accumulate (:2497-2536)
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

from . import (ACT_SWIGLU, DTYPE_BF16, DTYPE_F32, argmax, embedding, kv8, linear_workspace, q4_linear, rmsnorm,
               rmsnorm_mlp, rmsnorm_mlp_workspace, rmsnorm_qkv, rope)
from ._device import checked
from .qwen_decode import QWEN25_3B, Layer, QwenConfig, QwenQ4Decoder


class QwenKv8Decoder(QwenQ4Decoder):
    """`batch` sequences whose caches hold up to max_ctx tokens of `format` (kv8.INT8 or kv8.E4M3), the first `ctx` of them
    random as in QwenQ4Decoder.  Positions go on through evictions, up to max_positions."""

    def __init__(self, cfg: QwenConfig = QWEN25_3B, batch: int = 1, ctx: int = 512, seed: int = 3000,
                 device: str = "cuda", max_ctx: Optional[int] = None, format: int = kv8.INT8,
                 max_positions: Optional[int] = None, scaling: Optional[rope.Scaling] = None,
                 track_weights: bool = False):
        self._capacity = ctx + 1 if max_ctx is None else max_ctx
        if self._capacity < ctx:
            raise ValueError(f"max_ctx={max_ctx} is below ctx={ctx}")
        self._format, self._track = format, track_weights
        self.lengths = torch.full((batch,), ctx, dtype=torch.int32, device=device)
        super().__init__(cfg, batch, ctx, seed, device)
        positions = self._capacity if max_positions is None else max_positions
        self.cos_sin = rope.table(cfg.head_dim, positions, cfg.rope_theta, scaling=scaling, device=device)
        # tokens in the caches and next positions of the sequences, as far as the calls made here tell: a captured step's replays
        # move the device's alone
        self._used, self._next, self._captured = [ctx] * batch, [ctx] * batch, False
        self._spare = None
        self.attn = torch.empty((batch, cfg.q_heads, cfg.head_dim), dtype=torch.bfloat16, device=device)
        self.lse = torch.empty((batch, cfg.q_heads), dtype=torch.float32, device=device)
        self.attn_ws = kv8.attention_workspace(self.layers[0].cache, cfg.q_heads, batch)
        self.weight_ws = kv8.weight_workspace(self.layers[0].cache, cfg.q_heads, batch)
        self.o_ws = linear_workspace(batch, cfg.hidden, cfg.q_heads * cfg.head_dim, device=device)

    def _new_cache(self, device) -> kv8.Kv8Cache:
        c = self.cfg
        return kv8.Kv8Cache(self.batch, c.kv_heads, c.head_dim, self._capacity, format=self._format, device=device)

    def _new_weight(self, device) -> Optional[torch.Tensor]:
        shape = (self.batch, self.cfg.kv_heads, self._capacity)
        return torch.zeros(shape, dtype=torch.float32, device=device) if self._track else None

    def _placed(self, layer: Layer) -> Layer:
        rows = [t.flatten(0, 1) for t in (layer.k_cache, layer.v_cache)]  # ctx + 1 a sequence; the last one is cut off
        layer.cache, layer.weight = self._new_cache(rows[0].device), self._new_weight(rows[0].device)
        if self.ctx:
            first = torch.arange(rows[0].shape[0], device=rows[0].device).view(self.batch, -1)[:, : self.ctx].flatten()
            starts = torch.arange(0, (self.batch + 1) * self.ctx, self.ctx, dtype=torch.int32, device=rows[0].device)
            kv8.append(layer.cache, rows[0][first], rows[1][first], self.lengths, starts=starts)
        layer.k_cache = layer.v_cache = None
        return layer

    def _layers(self, h, x, qkv, attn, lse, positions, starts, attn_ws, weight_ws, o_ws, mlp_ws, stream):
        c, m = self.cfg, h.shape[0]
        q, k, v = (t.view(m, -1, c.head_dim) for t in qkv)
        for L in self.layers:
            rmsnorm_qkv(h, L.ln1, c.eps, L.q, L.k, L.v, q_bias=L.bq, k_bias=L.bk, v_bias=L.bv, out_dtype=DTYPE_BF16,
                        outs=qkv, xnorm=x, stream=stream)
            kv8.append(L.cache, k, v, self.lengths, starts=starts, q=q, cos_sin=self.cos_sin, positions=positions,
                       stream=stream)
            kv8.attention(L.cache, q, self.lengths, starts=starts, out=attn, lse=lse, workspace=attn_ws, stream=stream)
            if L.weight is not None:
                kv8.accumulate_weight(L.cache, q, lse, self.lengths, L.weight, starts=starts, workspace=weight_ws,
                                      stream=stream)
            q4_linear(L.o, attn, y=h, accumulate=True, workspace=o_ws, stream=stream)
            rmsnorm_mlp(L.gate, L.up, L.down, h, L.ln2, c.eps, activation=ACT_SWIGLU, workspace=mlp_ws, stream=stream)

    def _read_back(self, what: str) -> None:
        """The host's counts from the device's (a synchronization)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} reads lengths back: it cannot be part of a capture")
        self._used, self._next = torch.stack((self.lengths, self.positions)).tolist()

    def _grow(self, counts) -> None:
        used, after = ([a + n for a, n in zip(to, counts)] for to in (self._used, self._next))
        if max(used) > self._capacity:
            raise ValueError(f"a sequence of {max(used)} tokens exceeds max_ctx={self._capacity}: evict first")
        if max(after) > self.cos_sin.shape[0]:
            raise ValueError(f"position {max(after) - 1} has no row in the rotary table: max_positions={self.cos_sin.shape[0]}")
        self._used, self._next = used, after

    def step(self, stream=None) -> torch.Tensor:
        """One greedy decode step of every sequence: `tokens` are appended at `positions`, both move on; returns the
        next-token buffer.  stream: a torch.cuda.Stream.  Nothing returns to the host, so a step can be captured and replayed
        (as long as caches and rotary table hold: in replays keys that do not fit are cut off, positions past the table not
        turned).  Once a step has been captured, eager ones read the lengths back, to go by what replays have added."""
        with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
            if torch.cuda.is_current_stream_capturing():
                self._captured = True
            else:
                if self._captured:
                    self._read_back("an eager step")
                self._grow([1] * self.batch)
            self.lengths.add_(1)
            embedding(self.embed, self.tokens, out=self.h, stream=stream)
            self._layers(self.h, self.x, (self.q, self.k, self.v), self.attn, self.lse, self.positions, None,
                         self.attn_ws, self.weight_ws, self.o_ws, self.ws, stream)
            rmsnorm(self.h, self.ln_f, self.cfg.eps, out=self.x, stream=stream)
            q4_linear(self.embed, self.x, y=self.logits, out_dtype=DTYPE_F32, stream=stream)
            argmax(self.logits, out=self.next, workspace=self.argmax_ws, stream=stream)
            self.positions.add_(1)
        return self.next

    def prefill(self, tokens: torch.Tensor, counts) -> torch.Tensor:
        """Appends counts[b] tokens to each sequence b (tokens int32, sequence after sequence; a count may be 0) in one ragged
        batch and sets `logits` and `tokens` of those that got any to what follows their last one; returns the next-token buffer.
        Reads the lengths back, so it goes by what replays of a captured step have added too."""
        c, m, device = self.cfg, int(tokens.numel()), tokens.device
        counts = [int(n) for n in counts]
        if len(counts) != self.batch or min(counts) < 0 or sum(counts) != m:
            raise ValueError(f"counts={counts} do not split {m} tokens over {self.batch} sequences")
        if m == 0:
            return self.next
        checked("tokens", tokens, torch.int32, None, self.lengths)
        self._read_back("prefill")
        self._grow(counts)
        n = torch.tensor(counts, dtype=torch.int32, device=device)
        starts = torch.zeros(self.batch + 1, dtype=torch.int32, device=device)
        torch.cumsum(n, 0, dtype=torch.int32, out=starts[1:])
        place = torch.arange(m, dtype=torch.int32, device=device)
        seq = torch.repeat_interleave(torch.arange(self.batch, device=device), n, output_size=m)
        positions = self.positions[seq] + place - starts[seq]
        self.lengths.add_(n)

        def rows(width, dtype=torch.bfloat16):
            return torch.empty((m, width), dtype=dtype, device=device)
        qn, kn = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        h, x, qkv = rows(c.hidden), rows(c.hidden), (rows(qn), rows(kn), rows(kn))
        cache = self.layers[0].cache
        embedding(self.embed, tokens, out=h)
        self._layers(h, x, qkv, rows(qn).view(m, c.q_heads, c.head_dim), rows(c.q_heads, torch.float32), positions, starts,
                     kv8.attention_workspace(cache, c.q_heads, m), kv8.weight_workspace(cache, c.q_heads, m) if self._track else None,
                     linear_workspace(m, c.hidden, qn, device=device),
                     rmsnorm_mlp_workspace(m, c.hidden, c.inter, device=device), None)
        got = torch.tensor([b for b, n in enumerate(counts) if n], device=device)
        last = h[(starts[1:][got] - 1).long()].contiguous()
        last = rmsnorm(last, self.ln_f, c.eps)
        logits = q4_linear(self.embed, last, out_dtype=DTYPE_F32)
        self.logits[got] = logits
        self.tokens[got] = argmax(logits)
        self.positions.add_(n)
        return self.next

    def evict(self, budget: int, sink: int = 4, recent: int = 64) -> None:
        """Cuts every sequence's cache to `budget` tokens (kv8.evict): the first `sink`, the last `recent` and those of most
        attention weight since they were appended.  Needs track_weights.  Reads the lengths back; the layers' caches change places with a
        spare one: a captured step is to be captured again."""
        if not self._track:
            raise ValueError("evict needs a decoder with track_weights=True")
        self._read_back("evict")
        if self._spare is None:
            device = self.lengths.device
            self._spare = self._new_cache(device), self._new_weight(device)
        left = torch.empty_like(self.lengths)
        kept = torch.empty((self.batch, self.cfg.kv_heads, budget), dtype=torch.int32, device=left.device)
        for L in self.layers:
            cache, weight = self._spare
            kv8.evict(L.cache, self.lengths, L.weight, budget, sink, recent, cache, weight, kept, left)
            self._spare = L.cache, L.weight
            L.cache, L.weight = cache, weight
        self.lengths.copy_(left)
        self._used = [min(n, budget) for n in self._used]

