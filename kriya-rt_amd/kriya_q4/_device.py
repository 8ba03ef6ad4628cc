"""Checks of tensors, and the device and stream that a call on them runs on."""
from __future__ import annotations

import contextlib

import torch

_here = contextlib.nullcontext()
# torch.cuda.current_device() and current_stream() without the objects that they make: 2 us of a 4 us launch
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def at(t: torch.Tensor):
    """The device of t made current for a call (nothing to do where it is)."""
    return _here if t.get_device() == _device() else torch.cuda.device(t.device)


def stream_of(t: torch.Tensor, stream):
    """The raw stream of a call: the given one, else the current one of t's device."""
    if stream is None:
        return _raw_stream(t.get_device())
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def new(shape, dtype, device: torch.device, stream=None) -> torch.Tensor:
    """A tensor that a call on `stream` makes: of that stream's own memory, so that work still pending on the current stream never
    meets it and it is not reused before the call is done, and kept for the current stream, on which the caller goes on."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    here = torch.cuda.current_stream(device)
    raw = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
    if raw == here.cuda_stream:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(raw, device=here.device)):
        t = torch.empty(shape, dtype=dtype, device=here.device)
    t.record_stream(here)
    return t


def checked(name: str, t: torch.Tensor, dtype, shape=None, like=None) -> torch.Tensor:
    """t, after a check of its type, its shape (where one is given), its contiguity and its device."""
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, strides are {t.stride()}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, the other tensors on {like.device}")
    return t
