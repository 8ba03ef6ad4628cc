"""The 8-bit key/value cache (include/kriya_kv8.h): appending, attention over it from one token per sequence to whole
prompts, and the eviction of tokens by their accumulated attention weight.

A step over all layers shares `lengths` (int32 [batch]: the tokens of each sequence, this step's included) and, where
sequences have other than one new token, `starts` (int32 [batch + 1]: their rows in k, v and q)::

    cache = kv8.Kv8Cache(batch, kv_heads, head_dim, max_ctx)
    lengths += 1
    kv8.append(cache, k, v, lengths, q=q, q_out=q, cos_sin=table, positions=lengths - 1)
    out, lse = kv8.attention(cache, q, lengths)

Calls run on `stream` (a torch.cuda.Stream or a raw one), the current stream where None.  What a call allocates for itself or its
caller is of that stream's memory; inputs and given outputs are the caller's to order and to keep, as with any stream.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import DTYPE_BF16, DTYPE_F32, _check, lib
from . import rope as _rope
from ._device import at, checked, new, stream_of

INT8, E4M3 = 0, 1
BLOCK = 32
_BF16 = (torch.bfloat16,)


class kr_kv8_cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("k_open", ctypes.c_void_p), ("v_open", ctypes.c_void_p),
                ("batch", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("max_ctx", ctypes.c_uint32), ("format", ctypes.c_int)]


class Kv8Cache:
    """One layer's cache of `batch` sequences: bytes k, v uint8 [batch, kv_heads, blocks, 32 * head_dim], scales f32
    [batch, kv_heads, blocks], and the raw rows of each last block, bf16 [batch, kv_heads, 32, head_dim]."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, max_ctx: int, format: int = INT8, device="cuda"):
        blocks = -(-max_ctx // BLOCK)

        def new(dtype, *shape):
            return torch.empty((batch, kv_heads) + shape, dtype=dtype, device=device)
        self._hold(new(torch.uint8, blocks, BLOCK * head_dim), new(torch.uint8, blocks, BLOCK * head_dim),
                   new(torch.float32, blocks), new(torch.float32, blocks), new(torch.bfloat16, BLOCK, head_dim),
                   new(torch.bfloat16, BLOCK, head_dim), max_ctx, format)

    @classmethod
    def wrap(cls, k, v, k_scale, v_scale, k_open, v_open, max_ctx: int, format: int = INT8) -> "Kv8Cache":
        """A cache over tensors that the caller holds."""
        c = cls.__new__(cls)
        c._hold(k, v, k_scale, v_scale, k_open, v_open, max_ctx, format)
        return c

    def _hold(self, k, v, k_scale, v_scale, k_open, v_open, max_ctx, format):
        if k_open.dim() != 4:
            raise ValueError(f"k_open must be [batch, kv_heads, 32, head_dim], not {tuple(k_open.shape)}")
        b, h, _, d = k_open.shape
        blocks = -(-max_ctx // BLOCK)
        for name, t, dt, shape in (("k", k, torch.uint8, (b, h, blocks, BLOCK * d)),
                                   ("v", v, torch.uint8, (b, h, blocks, BLOCK * d)),
                                   ("k_scale", k_scale, torch.float32, (b, h, blocks)),
                                   ("v_scale", v_scale, torch.float32, (b, h, blocks)),
                                   ("k_open", k_open, torch.bfloat16, (b, h, BLOCK, d)),
                                   ("v_open", v_open, torch.bfloat16, (b, h, BLOCK, d))):
            checked(name, t, dt, shape, k)
        self.k, self.v, self.k_scale, self.v_scale, self.k_open, self.v_open = k, v, k_scale, v_scale, k_open, v_open
        self.batch, self.kv_heads, self.head_dim, self.max_ctx, self.format = b, h, d, max_ctx, format
        self._desc = kr_kv8_cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                  k_open.data_ptr(), v_open.data_ptr(), b, h, d, max_ctx, format)

    @property
    def desc(self):
        return ctypes.byref(self._desc)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_open, self.v_open))


def _step(cache: Kv8Cache, tokens: int, starts, lengths) -> Tuple[Optional[int], int]:
    checked("lengths", lengths, torch.int32, (cache.batch,), cache.k)
    if starts is None:
        return None, lengths.data_ptr()
    checked("starts", starts, torch.int32, (cache.batch + 1,), cache.k)
    return starts.data_ptr(), lengths.data_ptr()


def _same(t: torch.Tensor, like: torch.Tensor) -> bool:
    """Whether t has the type, shape, strides and device of a tensor that has been checked."""
    return (t is like or (t.dtype is like.dtype and t.shape == like.shape and t.stride() == like.stride()
                          and t.get_device() == like.get_device()))


def _queries(cache: Kv8Cache, q: torch.Tensor) -> int:
    stride = _rope.rows_of("q", q, _BF16, cache.k)
    if q.shape[2] != cache.head_dim:
        raise ValueError(f"q has head_dim {q.shape[2]}, the cache {cache.head_dim}")
    return stride


def append(cache: Kv8Cache, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor,
           starts: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
           q_out: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None, layout: int = _rope.HALF, stream=None) -> None:
    """Codes k, v (bf16 [tokens, kv_heads, head_dim]) into the last slots of their sequences; with cos_sin and positions,
    k is rotated first and q into q_out (q where None), all in one launch (kr_kv8_append)."""
    stride = _rope.rows_of("k", k, _BF16, cache.k)
    if not _same(v, k) and (v.dtype is not k.dtype or v.shape != k.shape or _rope.rows_of("v", v, _BF16, cache.k) != stride):
        raise ValueError("k and v must have the same type, shape and strides")
    tokens, heads, d = k.shape
    if heads != cache.kv_heads or d != cache.head_dim:
        raise ValueError(f"k must be [tokens, {cache.kv_heads}, {cache.head_dim}], not {tuple(k.shape)}")
    s, n = _step(cache, tokens, starts, lengths)
    r, qp, op, qs, heads = None, None, None, 0, 0
    if (cos_sin is None) != (positions is None):
        raise ValueError("cos_sin and positions go together")
    if cos_sin is not None:
        r = ctypes.byref(_rope.descriptor(cos_sin, positions, tokens, layout, False, cache.k))
    if q is not None:
        q_out = q if q_out is None else q_out
        qs, heads = _queries(cache, q), q.shape[1]
        if q.shape[0] != tokens or not (_same(q_out, q) or (q_out.shape == q.shape and _queries(cache, q_out) == qs)):
            raise ValueError("q and q_out must have the tokens of k, and the same shape and strides")
        qp, op = q.data_ptr(), q_out.data_ptr()
    with at(cache.k):
        _check(lib().kr_kv8_append(cache.desc, r, k.data_ptr(), v.data_ptr(), stride, qp, op, qs, heads, tokens, s, n,
                                   stream_of(cache.k, stream)))


def dequant(cache: Kv8Cache, lengths: torch.Tensor, count: int, first: Optional[torch.Tensor] = None,
            out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, dtype=torch.bfloat16, stream=None):
    """(k, v) [batch, count, kv_heads, head_dim]: what slots first[b] .. first[b] + count - 1 stand for, zeros from
    lengths[b] on (kr_kv8_dequant)."""
    shape = (cache.batch, count, cache.kv_heads, cache.head_dim)
    if out is None:
        out = new(shape, dtype, cache.k.device, stream), new(shape, dtype, cache.k.device, stream)
    else:
        checked("out[0]", out[0], out[0].dtype, shape, cache.k)
        checked("out[1]", out[1], out[0].dtype, shape, cache.k)
    if out[0].dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"dequant to {out[0].dtype}")
    _, n = _step(cache, 0, None, lengths)
    f = checked("first", first, torch.int32, (cache.batch,), cache.k).data_ptr() if first is not None else None
    with at(cache.k):
        _check(lib().kr_kv8_dequant(cache.desc, n, f, count, out[0].data_ptr(), out[1].data_ptr(),
                                    DTYPE_F32 if out[0].dtype == torch.float32 else DTYPE_BF16, stream_of(cache.k, stream)))
    return out


def attention_workspace(cache: Kv8Cache, q_heads: int, tokens: int, stream=None) -> torch.Tensor:
    """Device workspace of attention (partial sums of split contexts) for calls on `stream` (the current one where None); one
    made for a step serves all its layers."""
    n = int(lib().kr_kv8_attention_workspace_bytes(cache.desc, q_heads, tokens))
    return new((max(n, 16),), torch.uint8, cache.k.device, stream)


def attention(cache: Kv8Cache, q: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None,
              scale: Optional[float] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None, stream=None):
    """(out, lse) of q (bf16 [tokens, q_heads, head_dim]) over the cache, causal at its end: out bf16 like q, lse f32
    [tokens, q_heads] natural logarithms (kr_kv8_attention).  scale: 1 / sqrt(head_dim) where None."""
    qs = _queries(cache, q)
    tokens, heads, d = q.shape
    s, n = _step(cache, tokens, starts, lengths)
    if out is None:
        out = new((tokens, heads, d), torch.bfloat16, q.device, stream)
    if lse is None:
        lse = new((tokens, heads), torch.float32, q.device, stream)
    checked("out", out, torch.bfloat16, (tokens, heads, d), cache.k)
    checked("lse", lse, torch.float32, (tokens, heads), cache.k)
    if workspace is None:
        workspace = attention_workspace(cache, heads, tokens, stream)
    checked("workspace", workspace, torch.uint8, None, cache.k)
    with at(cache.k):
        _check(lib().kr_kv8_attention(cache.desc, q.data_ptr(), qs, heads, tokens, s, n,
                                      1.0 / math.sqrt(d) if scale is None else scale, out.data_ptr(), lse.data_ptr(),
                                      workspace.data_ptr(), workspace.numel(), stream_of(cache.k, stream)))
    return out, lse


def weight_workspace(cache: Kv8Cache, q_heads: int, tokens: int, stream=None) -> torch.Tensor:
    """Device workspace of accumulate_weight (sums of parts of many query rows) for calls on `stream`."""
    n = int(lib().kr_kv8_weight_workspace_bytes(cache.desc, q_heads, tokens))
    return new((max(n, 16),), torch.uint8, cache.k.device, stream)


def accumulate_weight(cache: Kv8Cache, q: torch.Tensor, lse: torch.Tensor, lengths: torch.Tensor, weight: torch.Tensor,
                      starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, decay: float = 1.0,
                      workspace: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """weight f32 [batch, kv_heads, max_ctx], in place: decay times what it holds, plus the attention weights that the
    tokens of q give each slot (kr_kv8_accumulate_weight); lse as attention returned it for this q."""
    qs = _queries(cache, q)
    tokens, heads, d = q.shape
    s, n = _step(cache, tokens, starts, lengths)
    checked("lse", lse, torch.float32, (tokens, heads), cache.k)
    checked("weight", weight, torch.float32, (cache.batch, cache.kv_heads, cache.max_ctx), cache.k)
    if workspace is None:
        workspace = weight_workspace(cache, heads, tokens, stream)
    checked("workspace", workspace, torch.uint8, None, cache.k)
    with at(cache.k):
        _check(lib().kr_kv8_accumulate_weight(cache.desc, q.data_ptr(), qs, heads, tokens, s, n,
                                              1.0 / math.sqrt(d) if scale is None else scale, lse.data_ptr(), decay,
                                              weight.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                              stream_of(cache.k, stream)))
    return weight


def evict(cache: Kv8Cache, lengths: torch.Tensor, weight: torch.Tensor, budget: int, sink: int, recent: int,
          to: Kv8Cache, to_weight: torch.Tensor, kept: Optional[torch.Tensor] = None,
          to_lengths: Optional[torch.Tensor] = None, stream=None):
    """Copies every sequence into the cache `to`, cut to `budget` tokens where it is longer: the first `sink`, the last
    `recent` and the heaviest between (kr_kv8_evict).  Returns (kept int32 [batch, kv_heads, budget], to_lengths
    int32 [batch])."""
    _, n = _step(cache, 0, None, lengths)
    if kept is None:
        kept = new((cache.batch, cache.kv_heads, budget), torch.int32, cache.k.device, stream)
    if to_lengths is None:
        to_lengths = new((cache.batch,), torch.int32, cache.k.device, stream)
    checked("to.k", to.k, torch.uint8, None, cache.k)
    checked("weight", weight, torch.float32, (cache.batch, cache.kv_heads, cache.max_ctx), cache.k)
    checked("to_weight", to_weight, torch.float32, (cache.batch, cache.kv_heads, to.max_ctx), cache.k)
    checked("kept", kept, torch.int32, (cache.batch, cache.kv_heads, budget), cache.k)
    checked("to_lengths", to_lengths, torch.int32, (cache.batch,), cache.k)
    with at(cache.k):
        _check(lib().kr_kv8_evict(cache.desc, n, weight.data_ptr(), budget, sink, recent, to.desc, to_weight.data_ptr(),
                                  kept.data_ptr(), to_lengths.data_ptr(), stream_of(cache.k, stream)))
    return kept, to_lengths
