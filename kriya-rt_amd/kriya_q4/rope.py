"""Rotary positions in general form (include/kriya_kv8.h): tables for stretched contexts, and the rotation of whole or
partial heads in either pairing, in place or not, inside the rows of a fused projection or not."""
from __future__ import annotations

import ctypes
import dataclasses
import math
from typing import Optional

import torch

from . import DTYPE_BF16, DTYPE_F32, KrError, KR_E_SHAPE, _check, lib
from ._device import at, checked, new, stream_of

HALF, INTERLEAVED = 0, 1
KINDS = {"none": 0, "linear": 1, "ntk": 2, "parts": 3}


class kr_rope_scaling(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int), ("factor", ctypes.c_double), ("original_ctx", ctypes.c_double),
                ("slow", ctypes.c_double), ("fast", ctypes.c_double), ("gain", ctypes.c_double)]


class kr_rope(ctypes.Structure):
    _fields_ = [("cos_sin", ctypes.c_void_p), ("positions", ctypes.c_void_p), ("rows", ctypes.c_uint32),
                ("rotary_dim", ctypes.c_uint32), ("layout", ctypes.c_int), ("inverse", ctypes.c_int)]


@dataclasses.dataclass(frozen=True)
class Scaling:
    """How the frequencies are stretched: "none", "linear" (position interpolation), "ntk" (a larger theta) or "parts"
    (by parts, between `slow` and `fast` turns over the trained context, as in the YaRN paper; checkpoints that ramp over the index of a
    frequency between whole numbers need a table made so, which every call here takes).  gain multiplies cos and sin; None takes 1,
    and 0.1 ln(factor) + 1 for "parts" with a factor above 1."""
    kind: str = "none"
    factor: float = 1.0
    original_ctx: float = 0.0
    slow: float = 1.0
    fast: float = 32.0
    gain: Optional[float] = None

    def _c(self) -> kr_rope_scaling:
        if self.kind not in KINDS:
            raise ValueError(f"scaling kind {self.kind!r} is not one of {sorted(KINDS)}")
        gain = self.gain
        if gain is None:
            gain = 0.1 * math.log(self.factor) + 1.0 if self.kind == "parts" and self.factor > 1.0 else 1.0
        return kr_rope_scaling(KINDS[self.kind], self.factor, self.original_ctx, self.slow, self.fast, gain)


def table(rotary_dim: int, count: int, theta: float, first: int = 0, scaling: Optional[Scaling] = None,
          out: Optional[torch.Tensor] = None, device="cuda", stream=None) -> torch.Tensor:
    """cos and sin of positions first .. first + count - 1: f32 [count, rotary_dim / 2, 2] (kr_rope_table)."""
    if out is None:
        out = new((count, rotary_dim // 2, 2), torch.float32, torch.device(device), stream)
    checked("out", out, torch.float32, (count, rotary_dim // 2, 2))
    z = ctypes.byref(scaling._c()) if scaling is not None else None
    with at(out):
        _check(lib().kr_rope_table(out.data_ptr(), first, count, rotary_dim, theta, z, stream_of(out, stream)))
    return out


def descriptor(cos_sin: torch.Tensor, positions: torch.Tensor, tokens: int, layout: int = HALF,
               inverse: bool = False, like: Optional[torch.Tensor] = None) -> kr_rope:
    """kr_rope of a table f32 [rows, rotary_dim / 2, 2] and int32 positions [tokens]."""
    if cos_sin.dim() != 3 or cos_sin.shape[2] != 2:
        raise ValueError(f"cos_sin must be [rows, rotary_dim / 2, 2], not {tuple(cos_sin.shape)}")
    checked("cos_sin", cos_sin, torch.float32, None, like)
    checked("positions", positions, torch.int32, (tokens,), like)
    return kr_rope(cos_sin.data_ptr(), positions.data_ptr(), cos_sin.shape[0], 2 * cos_sin.shape[1], layout, int(inverse))


def rows_of(name: str, t: torch.Tensor, dtypes, like: Optional[torch.Tensor] = None) -> int:
    """The token stride of t [tokens, heads, head_dim], whose heads lie side by side."""
    if t.dim() != 3 or t.dtype not in dtypes:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] of {dtypes}, not {tuple(t.shape)} of {t.dtype}")
    if not t.is_cuda or (like is not None and t.get_device() != like.get_device()):
        raise ValueError(f"{name} must be on the same GPU as the other tensors")
    tokens, heads, d = t.shape
    s0, s1, s2 = t.stride()
    if (d > 1 and s2 != 1) or (heads > 1 and s1 != d):
        raise ValueError(f"{name}: the heads of a token must be contiguous, strides are {t.stride()}")
    stride = s0 if tokens > 1 else max(heads * d, 1)
    if tokens > 1 and stride < heads * d:
        raise KrError(KR_E_SHAPE, f"{name}: tokens overlap, strides are {t.stride()}")
    return stride


def apply(x: torch.Tensor, cos_sin: torch.Tensor, positions: torch.Tensor, layout: int = HALF, inverse: bool = False,
          out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [tokens, heads, head_dim] (bf16 or f32; tokens may be strided) rotated to its positions, in place or into `out`
    (kr_rope_apply).  inverse: by the negative angles, which is also the gradient of the rotation."""
    if out is None:
        out = x
    xs = rows_of("x", x, (torch.bfloat16, torch.float32))
    ys = rows_of("out", out, (x.dtype,), x)
    if out.shape != x.shape:
        raise ValueError(f"out is {tuple(out.shape)}, x {tuple(x.shape)}")
    tokens, heads, d = x.shape
    r = descriptor(cos_sin, positions, tokens, layout, inverse, x)
    with at(x):
        _check(lib().kr_rope_apply(ctypes.byref(r), x.data_ptr(), xs, out.data_ptr(), ys,
                                   DTYPE_F32 if x.dtype == torch.float32 else DTYPE_BF16, tokens, heads, d,
                                   stream_of(x, stream)))
    return out
