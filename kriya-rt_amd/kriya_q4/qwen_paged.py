"""The Qwen2.5-shaped decoder of kriya_q4.qwen_decode over a cache in pages that its sequences share: prompts as ragged batches,
decoding, the verification of drafted trees, and sequences that end and make room for others.

A layer is that of qwen_decode, with its attention block in these calls:

    q, k, v = rmsnorm(h, ln1) Wq^T + bq, ...           encode_fused_qkv (encoder.rs:2539-2619)
    rope(q, k) at the positions; k, v into the pages   paged.append, one launch
    a = attention(q, K, V)                             paged.attention, causal or by the trees' masks
    h += a Wo^T                                        encode_q4_linear_accumulate (:2497-2536)
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

from . import (ACT_SWIGLU, DTYPE_BF16, DTYPE_F32, argmax, embedding, linear_workspace, paged, q4_linear, rmsnorm, rmsnorm_mlp,
               rmsnorm_mlp_workspace, rmsnorm_qkv, rope)
from ._device import checked
from .qwen_decode import QWEN25_3B, Layer, QwenConfig, QwenQ4Decoder


class QwenPagedDecoder(QwenQ4Decoder):
    """`batch` sequences of up to max_ctx tokens over a pool of `pages` pages (as many as they could all fill where None), the first
    `ctx` tokens random as in QwenQ4Decoder.  Eager calls take pages from the pool as sequences grow; replays of a captured step
    need theirs before (reserve): what they add beyond is lost, and the next eager calls are refused until that sequence is released.  A released sequence takes no part in
    steps, eager or replayed (its rows of `tokens` and `logits` mean nothing), until a prompt or a tree fills its place.  A prompt or a tree counts once all of
    its pass has been enqueued: a call that is refused or fails leaves the sequences as they were.  All calls on one stream, or
    ordered by the caller."""

    def __init__(self, cfg: QwenConfig = QWEN25_3B, batch: int = 1, ctx: int = 512, seed: int = 3000,
                 device: str = "cuda", max_ctx: Optional[int] = None, page: int = 64, pages: Optional[int] = None,
                 scaling: Optional[rope.Scaling] = None):
        self._capacity = ctx + 1 if max_ctx is None else max_ctx
        if self._capacity < ctx:
            raise ValueError(f"max_ctx={max_ctx} is below ctx={ctx}")
        most = -(-self._capacity // page)
        self.cache = paged.PagedCache(cfg.layers, batch * most if pages is None else pages, page, cfg.kv_heads, cfg.head_dim, device)
        self._free = list(range(self.cache.pages))[::-1]
        self._pages = [[] for _ in range(batch)]
        self.table = torch.full((batch, most), -1, dtype=torch.int32, device=device)
        # tokens in the pages, as far as the calls made here tell: replays of a captured step move the device's alone
        self._used, self._captured = [ctx] * batch, False
        # 1 of sequences that take part in steps, on the device, where replays read it, and here
        self.active, self._active = torch.ones(batch, dtype=torch.int32, device=device), [1] * batch
        self.lengths = torch.full((batch,), ctx, dtype=torch.int32, device=device)
        self._take([ctx] * batch)
        super().__init__(cfg, batch, ctx, seed, device)
        self.cos_sin = rope.table(cfg.head_dim, self._capacity, cfg.rope_theta, scaling=scaling, device=device)
        self._step = paged.Step(self.table, self.lengths)
        self.attn = torch.empty((batch, cfg.q_heads, cfg.head_dim), dtype=torch.bfloat16, device=device)
        self.lse = torch.empty((batch, cfg.q_heads), dtype=torch.float32, device=device)
        self.attn_ws = paged.attention_workspace(self.cache, self._step, cfg.q_heads, batch)
        self.o_ws = linear_workspace(batch, cfg.hidden, cfg.q_heads * cfg.head_dim, device=device)

    def _placed(self, layer: Layer) -> Layer:
        rows = [t.flatten(0, 1) for t in (layer.k_cache, layer.v_cache)]  # ctx + 1 a sequence; the last one is cut off
        if self.ctx:
            first = torch.arange(rows[0].shape[0], device=rows[0].device).view(self.batch, -1)[:, : self.ctx].flatten()
            starts = torch.arange(0, (self.batch + 1) * self.ctx, self.ctx, dtype=torch.int32, device=rows[0].device)
            paged.append(self.cache, paged.Step(self.table, self.lengths, starts), rows[0][first], rows[1][first], len(self.layers))
        layer.k_cache = layer.v_cache = None
        return layer

    def _take(self, after) -> None:
        """Pages for sequences of `after` tokens, or an error before anything has changed."""
        if max(after) > self._capacity:
            raise ValueError(f"a sequence of {max(after)} tokens exceeds max_ctx={self._capacity}")
        need = [max(-(-n // self.cache.page) - len(have), 0) for n, have in zip(after, self._pages)]
        if sum(need) > len(self._free):
            raise ValueError(f"{sum(need)} pages are needed, {len(self._free)} of {self.cache.pages} are free: release sequences first")
        for b, n in enumerate(need):
            if n:
                new, have = [self._free.pop() for _ in range(n)], len(self._pages[b])
                self.table[b, have: have + n] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
                self._pages[b] += new

    def _read_back(self, what: str, past: bool = False) -> None:
        """The host's counts from the device's (a synchronization).  past: they may be past the sequences' pages."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} counts pages on the host: it cannot be part of a capture")
        used = self.lengths.tolist()
        for b, n in enumerate(used):
            if n > self.cache.page * len(self._pages[b]) and not past:
                raise RuntimeError(f"replays have brought sequence {b} to {n} tokens, past its {len(self._pages[b])} pages: reserve before "
                                   "them; now it can only be released")
        self._used = used

    def _grow(self, counts) -> None:
        after = [a + n for a, n in zip(self._used, counts)]
        self._take(after)
        self._used = after

    def reserve(self, tokens: int) -> None:
        """Gives every sequence that has not ended the pages for `tokens` more: what so many replays of a captured step need.  Reads the
        lengths back."""
        self._read_back("reserve")
        self._take([n + tokens * live for n, live in zip(self._used, self._active)])

    def release(self, sequence: int) -> None:
        """Ends a sequence: its pages are free for others, its length is 0 and stays so.  Reads the lengths back."""
        if not 0 <= sequence < self.batch:
            raise ValueError(f"sequence={sequence} is not 0 .. {self.batch - 1}")
        self._read_back("release", past=True)
        self._free += self._pages[sequence][::-1]
        self._pages[sequence] = []
        self.table[sequence].fill_(-1)
        for t in (self.lengths, self.positions, self.active):
            t[sequence: sequence + 1].zero_()
        self._used[sequence] = self._active[sequence] = 0

    def _layers(self, h, x, qkv, attn, lse, step, positions, mask, attn_ws, o_ws, mlp_ws, stream):
        c, m = self.cfg, h.shape[0]
        q, k, v = (t.view(m, -1, c.head_dim) for t in qkv)
        for i, L in enumerate(self.layers):
            rmsnorm_qkv(h, L.ln1, c.eps, L.q, L.k, L.v, q_bias=L.bq, k_bias=L.bk, v_bias=L.bv, out_dtype=DTYPE_BF16,
                        outs=qkv, xnorm=x, stream=stream)
            paged.append(self.cache, step, k, v, i, q=q, cos_sin=self.cos_sin, positions=positions, stream=stream)
            paged.attention(self.cache, step, q, i, mask=mask, out=attn, lse=lse, workspace=attn_ws, stream=stream)
            q4_linear(L.o, attn, y=h, accumulate=True, workspace=o_ws, stream=stream)
            rmsnorm_mlp(L.gate, L.up, L.down, h, L.ln2, c.eps, activation=ACT_SWIGLU, workspace=mlp_ws, stream=stream)

    def step(self, stream=None) -> torch.Tensor:
        """One greedy decode step of every sequence that has not ended: `tokens` are appended at `positions`, both move on; returns the
        next-token buffer.  stream: a torch.cuda.Stream.  Nothing returns to the host, so a step can be captured and replayed; once one has been,
        eager ones read the lengths back first."""
        with torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext():
            if torch.cuda.is_current_stream_capturing():
                self._captured = True
            else:
                if self._captured:
                    self._read_back("an eager step")
                self._grow(self._active)
            # (one that has ended stays at 0 tokens, its new one without a slot: nothing is appended, and its row sees nothing)
            self.lengths.add_(self.active)
            embedding(self.embed, self.tokens, out=self.h, stream=stream)
            self._layers(self.h, self.x, (self.q, self.k, self.v), self.attn, self.lse, self._step, self.positions, None,
                         self.attn_ws, self.o_ws, self.ws, stream)
            rmsnorm(self.h, self.ln_f, self.cfg.eps, out=self.x, stream=stream)
            q4_linear(self.embed, self.x, y=self.logits, out_dtype=DTYPE_F32, stream=stream)
            argmax(self.logits, out=self.next, workspace=self.argmax_ws, stream=stream)
            self.positions.add_(self.active)
        return self.next

    def _ragged(self, tokens: torch.Tensor, counts, what: str):
        """A ragged batch: counts, starts and the lengths after it on the device, after pages for it have been taken."""
        m, device = int(tokens.numel()), self.lengths.device
        counts = [int(n) for n in counts]
        if len(counts) != self.batch or min(counts) < 0 or sum(counts) != m:
            raise ValueError(f"counts={counts} do not split {m} tokens over {self.batch} sequences")
        if m:
            checked("tokens", tokens, torch.int32, None, self.lengths)
        self._read_back(what)
        self._take([a + n for a, n in zip(self._used, counts)])
        n = torch.tensor(counts, dtype=torch.int32, device=device)
        starts = torch.zeros(self.batch + 1, dtype=torch.int32, device=device)
        torch.cumsum(n, 0, dtype=torch.int32, out=starts[1:])
        return counts, n, starts, self.lengths + n

    def _counted(self, counts, lengths, used) -> None:
        """A ragged batch is part of its sequences."""
        self.lengths.copy_(lengths)
        self._used = used
        for b, n in enumerate(counts):
            if n and not self._active[b]:
                self.active[b: b + 1].fill_(1)
                self._active[b] = 1

    def _hidden(self, tokens, step, positions, mask) -> torch.Tensor:
        """The last layer's output of a ragged batch."""
        c, m, device = self.cfg, int(tokens.numel()), tokens.device

        def rows(width, dtype=torch.bfloat16):
            return torch.empty((m, width), dtype=dtype, device=device)
        qn, kn = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        h, x, qkv = rows(c.hidden), rows(c.hidden), (rows(qn), rows(kn), rows(kn))
        embedding(self.embed, tokens, out=h)
        self._layers(h, x, qkv, rows(qn).view(m, c.q_heads, c.head_dim), rows(c.q_heads, torch.float32), step, positions, mask,
                     paged.attention_workspace(self.cache, step, c.q_heads, m), linear_workspace(m, c.hidden, qn, device=device),
                     rmsnorm_mlp_workspace(m, c.hidden, c.inter, device=device), None)
        return h

    def prefill(self, tokens: torch.Tensor, counts) -> torch.Tensor:
        """Appends counts[b] tokens to each sequence b (tokens int32, sequence after sequence; a count may be 0) in one ragged
        batch and sets `logits` and `tokens` of those that got any to what follows their last one; returns the next-token buffer.
        Reads the lengths back."""
        counts, n, starts, after = self._ragged(tokens, counts, "prefill")
        m = int(tokens.numel())
        if m == 0:
            return self.next
        place = torch.arange(m, dtype=torch.int32, device=tokens.device)
        seq = torch.repeat_interleave(torch.arange(self.batch, device=tokens.device), n, output_size=m)
        positions = self.positions[seq] + place - starts[seq]
        h = self._hidden(tokens, paged.Step(self.table, after, starts), positions, None)
        got = torch.tensor([b for b, n in enumerate(counts) if n], device=tokens.device)
        last = rmsnorm(h[(starts[1:][got] - 1).long()].contiguous(), self.ln_f, self.cfg.eps)
        logits = q4_linear(self.embed, last, out_dtype=DTYPE_F32)
        chosen = argmax(logits)
        self.logits[got] = logits
        self.tokens[got] = chosen
        self.positions.add_(n)
        self._counted(counts, after, [a + n for a, n in zip(self._used, counts)])
        return self.next

    def verify(self, tokens: torch.Tensor, parents: torch.Tensor, counts):
        """One pass over counts[b] drafted tokens of each sequence b (int32, sequence after sequence; a count may be 0): trees, by
        each node's parent among its sequence's nodes; node 0 is the sequence's entry of `tokens`, parent -1.  Keeps the path on which
        the drafts are the model's greedy choices and sets `logits` and `tokens` to what follows it, as that many steps would have.
        Returns (path int32 [batch, most nodes], counts int32 [batch]): the nodes kept.  Reads the lengths back."""
        if parents.shape != tokens.shape:
            raise ValueError(f"parents must be {tuple(tokens.shape)} like tokens, not {tuple(parents.shape)}")
        if tokens.numel():
            checked("tokens", tokens, torch.int32, (tokens.numel(),), self.lengths)
            checked("parents", parents, torch.int32, (tokens.numel(),), self.lengths)
        counts = [int(n) for n in counts]
        most = max(counts, default=0)
        if most > paged.MAX_NODES:
            raise ValueError(f"a tree of {most} nodes, more than {paged.MAX_NODES}")
        counts, n, starts, after = self._ragged(tokens, counts, "verify")
        if most == 0:
            return torch.zeros((self.batch, 1), dtype=torch.int32, device=n.device), torch.zeros_like(n)
        step = paged.Step(self.table, after, starts)
        mask, positions = paged.tree_plan(parents, after, starts, nodes=most)
        h = rmsnorm(self._hidden(tokens, step, positions, mask), self.ln_f, self.cfg.eps)
        logits = q4_linear(self.embed, h, out_dtype=DTYPE_F32)
        # (its next tokens beside `tokens`, which may be the nodes of this tree)
        path, kept, chosen, lengths = paged.commit(self.cache, step, tokens, parents, argmax(logits), next=self.tokens.clone(), max_path=most)
        got = torch.tensor([b for b, n in enumerate(counts) if n], device=n.device)
        self.logits[got] = logits[starts[:-1][got].long() + path[got, (kept[got] - 1).long()].long()]
        self.tokens.copy_(chosen)
        self.positions.copy_(lengths)
        self._counted(counts, lengths, lengths.tolist())
        return path, kept
