"""The paged key/value cache (include/kriya_paged.h): one pool of pages for all sequences and layers, appending with the heads'
norm and rotation, attention from one token per sequence to whole prompts and trees of drafted tokens, and the plan and
commit of such trees.

A step shares its sequences over all layers: the page table (int32 [batch, max_pages]; -1: no page), `lengths` (int32 [batch]:
the tokens of each sequence, this step's included) and, where sequences have other than one new token, `starts` (int32
[batch + 1]: their rows in k, v and q)::

    cache = paged.PagedCache(layers, pages, page, kv_heads, head_dim)
    step = paged.Step(table, lengths, starts)
    mask, positions = paged.tree_plan(parents, lengths, starts, nodes=64)
    for layer in range(layers):
        paged.append(cache, step, k, v, layer, q=q, cos_sin=cos_sin, positions=positions)
        out, lse = paged.attention(cache, step, q, layer, mask=mask)
    path, counts, next, lengths = paged.commit(cache, step, tokens, parents, targets)

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

UNIT = 16
MAX_NODES = 4096  # of a sequence's tree
_BF16 = (torch.bfloat16,)


class kr_paged_cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("layers", ctypes.c_uint32), ("pages", ctypes.c_uint32),
                ("page", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32)]


class kr_paged_step(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("max_pages", ctypes.c_uint32), ("batch", ctypes.c_uint32),
                ("starts", ctypes.c_void_p), ("lengths", ctypes.c_void_p)]


class kr_head_norm(ctypes.Structure):
    _fields_ = [("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p), ("eps", ctypes.c_float)]


class PagedCache:
    """The pool: k, v bf16 [layers, pages, kv_heads, page // 16, 16 * head_dim], units of 16 slots in the order of
    include/kriya_paged.h (read gives rows back)."""

    def __init__(self, layers: int, pages: int, page: int, kv_heads: int, head_dim: int, device="cuda"):
        if page < UNIT or page % UNIT:
            raise ValueError(f"page={page} is not a multiple of {UNIT}")
        shape = (layers, pages, kv_heads, page // UNIT, UNIT * head_dim)
        self._hold(*(torch.empty(shape, dtype=torch.bfloat16, device=device) for _ in "kv"))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedCache":
        """A pool over tensors that the caller holds."""
        c = cls.__new__(cls)
        c._hold(k, v)
        return c

    def _hold(self, k, v):
        if k.dim() != 5 or k.shape[4] % UNIT:
            raise ValueError(f"k must be [layers, pages, kv_heads, page / 16, 16 * head_dim], not {tuple(k.shape)}")
        checked("k", k, torch.bfloat16)
        checked("v", v, torch.bfloat16, k.shape, k)
        self.k, self.v = k, v
        self.layers, self.pages, self.kv_heads = k.shape[:3]
        self.page, self.head_dim = UNIT * k.shape[3], k.shape[4] // UNIT
        self._desc = kr_paged_cache(k.data_ptr(), v.data_ptr(), self.layers, self.pages, self.page, self.kv_heads, self.head_dim)
        self._ref = ctypes.byref(self._desc)

    @property
    def desc(self):
        return self._ref

    def nbytes(self) -> int:
        return 2 * self.k.numel() * self.k.element_size()


class Step:
    """The sequences of a step: their pages, lengths and new tokens' rows.  Holds the tensors; their contents may change from call to
    call."""

    def __init__(self, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None):
        if table.dim() != 2:
            raise ValueError(f"table must be [batch, max_pages], not {tuple(table.shape)}")
        checked("table", table, torch.int32)
        checked("lengths", lengths, torch.int32, table.shape[:1], table)
        if starts is not None:
            checked("starts", starts, torch.int32, (table.shape[0] + 1,), table)
        self.table, self.lengths, self.starts = table, lengths, starts
        self.batch, self.max_pages = table.shape
        self._desc = kr_paged_step(table.data_ptr(), self.max_pages, self.batch, None if starts is None else starts.data_ptr(),
                                   lengths.data_ptr())
        self._ref = ctypes.byref(self._desc)

    @property
    def desc(self):
        return self._ref


def _together(cache: PagedCache, step: Step) -> None:
    if step.table.get_device() != cache.k.get_device():
        raise ValueError(f"the step is on {step.table.device}, the cache on {cache.k.device}")


def _heads(cache: PagedCache, name: str, x: torch.Tensor) -> int:
    stride = _rope.rows_of(name, x, _BF16, cache.k)
    if x.shape[2] != cache.head_dim:
        raise ValueError(f"{name} has head_dim {x.shape[2]}, the cache {cache.head_dim}")
    return stride


def _alike(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether what holds for y holds for x: quicker than the checks again (0.3 us of a call of 9)."""
    return x.shape == y.shape and x.stride() == y.stride() and x.dtype is y.dtype and x.get_device() == y.get_device()


def append(cache: PagedCache, step: Step, k: torch.Tensor, v: torch.Tensor, layer: int = 0, q: Optional[torch.Tensor] = None,
           q_out: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None, layout: int = _rope.HALF, q_norm: Optional[torch.Tensor] = None,
           k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, stream=None) -> None:
    """Puts k, v (bf16 [tokens, kv_heads, head_dim]) into the pages of their sequences' last slots; with k_norm, q_norm (bf16
    [head_dim]) heads are normalised first, with cos_sin and positions rotated; q goes into q_out (q where None).  One launch
    (kr_paged_append)."""
    _together(cache, step)
    stride = _heads(cache, "k", k)
    if not _alike(v, k) and (v.shape != k.shape or _heads(cache, "v", v) != stride):
        raise ValueError("k and v must have the same shape and strides")
    tokens, heads, d = k.shape
    if heads != cache.kv_heads:
        raise ValueError(f"k must be [tokens, {cache.kv_heads}, {cache.head_dim}], not {tuple(k.shape)}")
    if (cos_sin is None) != (positions is None):
        raise ValueError("cos_sin and positions go together")
    r = n = qp = op = None
    qs = q_heads = 0
    if cos_sin is not None:
        r = ctypes.byref(_rope.descriptor(cos_sin, positions, tokens, layout, False, cache.k))
    if q_norm is not None or k_norm is not None:
        weights = [None if w is None else checked(name, w, torch.bfloat16, (d,), cache.k).data_ptr()
                   for name, w in (("q_norm", q_norm), ("k_norm", k_norm))]
        n = ctypes.byref(kr_head_norm(weights[0], weights[1], eps))
    if q is not None:
        q_out = q if q_out is None else q_out
        qs, q_heads = _heads(cache, "q", q), q.shape[1]
        if q.shape[0] != tokens or (not _alike(q_out, q) and (q_out.shape != q.shape or _heads(cache, "q_out", q_out) != qs)):
            raise ValueError("q and q_out must have the tokens of k, and the same shape and strides")
        qp, op = q.data_ptr(), q_out.data_ptr()
    with at(cache.k):
        _check(lib().kr_paged_append(cache.desc, layer, step.desc, n, r, k.data_ptr(), v.data_ptr(), stride, qp, op, qs, q_heads,
                                     tokens, stream_of(cache.k, stream)))


def read(cache: PagedCache, step: Step, count: int, layer: int = 0, first: Optional[torch.Tensor] = None, dtype=torch.bfloat16,
         out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, stream=None):
    """(k, v) [batch, count, kv_heads, head_dim]: slots first[b] .. first[b] + count - 1, zeros from lengths[b] on (kr_paged_read)."""
    _together(cache, step)
    shape = (step.batch, count, cache.kv_heads, cache.head_dim)
    if out is None:
        out = new(shape, dtype, cache.k.device, stream), new(shape, dtype, cache.k.device, stream)
    else:
        checked("out[0]", out[0], out[0].dtype, shape, cache.k)
        checked("out[1]", out[1], out[0].dtype, shape, cache.k)
    if out[0].dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"read into {out[0].dtype}")
    f = checked("first", first, torch.int32, (step.batch,), cache.k).data_ptr() if first is not None else None
    with at(cache.k):
        _check(lib().kr_paged_read(cache.desc, layer, step.desc, f, count, out[0].data_ptr(), out[1].data_ptr(),
                                   DTYPE_F32 if out[0].dtype == torch.float32 else DTYPE_BF16, stream_of(cache.k, stream)))
    return out


def attention_workspace(cache: PagedCache, step: Step, q_heads: int, tokens: int, stream=None) -> torch.Tensor:
    """Device workspace of attention (partial sums of split contexts) for calls on `stream`; one made for a step serves all its
    layers."""
    n = int(lib().kr_paged_attention_workspace_bytes(cache.desc, step.desc, q_heads, tokens))
    return new((max(n, 16),), torch.uint8, cache.k.device, stream)


def attention(cache: PagedCache, step: Step, q: torch.Tensor, layer: int = 0, mask: Optional[torch.Tensor] = None,
              scale: Optional[float] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None, stream=None):
    """(out, lse) of q (bf16 [tokens, q_heads, head_dim]) over the sequences' pages: out bf16 like q, lse f32 [tokens, q_heads]
    natural logarithms (kr_paged_attention).  Causal at each sequence's end, or, with mask (int32 [tokens, words], bit j of a row:
    the token sees its sequence's j-th new token), over the tokens before the step and those.  scale: 1 / sqrt(head_dim) where
    None."""
    _together(cache, step)
    qs = _heads(cache, "q", q)
    tokens, heads, d = q.shape
    words, mp = 0, None
    if mask is not None:
        if mask.dim() != 2 or mask.shape[0] != tokens:
            raise ValueError(f"mask must be [{tokens}, words], not {tuple(mask.shape)}")
        words, mp = mask.shape[1], checked("mask", mask, torch.int32, None, cache.k).data_ptr()
        if words == 0 and tokens:
            raise ValueError("mask has no words")
    if out is None:
        out = new((tokens, heads, d), torch.bfloat16, q.device, stream)
    if lse is None:
        lse = new((tokens, heads), torch.float32, q.device, stream)
    checked("out", out, torch.bfloat16, (tokens, heads, d), cache.k)
    checked("lse", lse, torch.float32, (tokens, heads), cache.k)
    if workspace is None:
        workspace = attention_workspace(cache, step, heads, tokens, stream)
    checked("workspace", workspace, torch.uint8, None, cache.k)
    with at(cache.k):
        _check(lib().kr_paged_attention(cache.desc, layer, step.desc, q.data_ptr(), qs, heads, tokens, mp, words,
                                        1.0 / math.sqrt(d) if scale is None else scale, out.data_ptr(), lse.data_ptr(),
                                        workspace.data_ptr(), workspace.numel(), stream_of(cache.k, stream)))
    return out, lse


def tree_plan(parents: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, nodes: Optional[int] = None,
              mask: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, stream=None):
    """(mask int32 [tokens, words], positions int32 [tokens]) of the trees of drafted tokens: the bits of each node's ancestors and
    its own, and its position (kr_tree_plan).  parents int32 [tokens]: the place of a node's parent among its sequence's nodes, -1
    for none.  nodes: the most of a sequence, which gives the words of a new mask."""
    tokens, batch = parents.shape[0], lengths.shape[0]
    checked("parents", parents, torch.int32, (tokens,))
    checked("lengths", lengths, torch.int32, (batch,), parents)
    s = checked("starts", starts, torch.int32, (batch + 1,), parents).data_ptr() if starts is not None else None
    if mask is None:
        if nodes is None or nodes < 1:
            raise ValueError("a new mask needs the most nodes of a sequence")
        mask = new((tokens, -(-nodes // 32)), torch.int32, parents.device, stream)
    if positions is None:
        positions = new((tokens,), torch.int32, parents.device, stream)
    if mask.dim() != 2:
        raise ValueError(f"mask must be [{tokens}, words], not {tuple(mask.shape)}")
    checked("mask", mask, torch.int32, (tokens, mask.shape[1]), parents)
    checked("positions", positions, torch.int32, (tokens,), parents)
    with at(parents):
        _check(lib().kr_tree_plan(parents.data_ptr(), tokens, s, lengths.data_ptr(), batch, mask.shape[1], mask.data_ptr(),
                                  positions.data_ptr(), stream_of(parents, stream)))
    return mask, positions


def commit(cache: PagedCache, step: Step, tokens: torch.Tensor, parents: torch.Tensor, targets: torch.Tensor,
           path: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None, next: Optional[torch.Tensor] = None,
           new_lengths: Optional[torch.Tensor] = None, max_path: Optional[int] = None, stream=None):
    """(path int32 [batch, max_path], counts, next, new_lengths int32 [batch]): the path that each sequence's tree shares with the
    model's choices (targets int32 [tokens]: after each node), its keys and values moved behind the sequence's tokens in all layers,
    the choice after it and the new length (kr_paged_commit).  max_path: 32 where neither it nor path is given.  A sequence without
    new tokens keeps what `next` held (0 in a new one)."""
    _together(cache, step)
    rows = tokens.shape[0]
    for name, t in (("tokens", tokens), ("parents", parents), ("targets", targets)):
        checked(name, t, torch.int32, (rows,), cache.k)
    device = cache.k.device
    if path is None:
        path = new((step.batch, 32 if max_path is None else max_path), torch.int32, device, stream)
    if path.dim() != 2 or (max_path is not None and path.shape[1] != max_path):
        raise ValueError(f"path must be [batch, max_path], not {tuple(path.shape)}")
    checked("path", path, torch.int32, (step.batch, path.shape[1]), cache.k)
    if counts is None:
        counts = new((step.batch,), torch.int32, device, stream)
    if next is None:
        next = new((step.batch,), torch.int32, device, stream, zero=True)
    if new_lengths is None:
        new_lengths = new((step.batch,), torch.int32, device, stream)
    for name, t in (("counts", counts), ("next", next), ("new_lengths", new_lengths)):
        checked(name, t, torch.int32, (step.batch,), cache.k)
    with at(cache.k):
        _check(lib().kr_paged_commit(cache.desc, step.desc, tokens.data_ptr(), parents.data_ptr(), targets.data_ptr(), rows,
                                     path.shape[1], path.data_ptr(), counts.data_ptr(), next.data_ptr(), new_lengths.data_ptr(),
                                     stream_of(cache.k, stream)))
    return path, counts, next, new_lengths
