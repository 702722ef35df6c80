"""Argument checks and pointer/stream extraction shared by the Python entry points.

The reference relies on trace-time ``assert``s and otherwise launches blindly
(python/cutedsl_kernels/gemm/kernel/attempt4.py:69,80-82,121,130). Here every
entry point checks dtype, device, shape and contiguity before it launches and
raises ``TypeError`` (wrong dtype / not a tensor) or ``ValueError`` (shape,
device, layout); the C ABI re-checks sizes and alignment.
"""
from __future__ import annotations

import torch

from . import _native


def require_tensor(name: str, t, dtype: torch.dtype, ndim: int | None = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (row-major)")
    return t


def require_shape(name: str, t: torch.Tensor, shape: tuple) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def same_device(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts[1:]:
        if t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    return dev


def stream_for(dev: torch.device, stream=None) -> int:
    """cudaStream_t (as int) to launch on: explicit, else torch's current stream."""
    _native.use_device(dev.index if dev.index is not None else torch.cuda.current_device())
    if stream is None:
        return torch.cuda.current_stream(dev).cuda_stream
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


_DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1}  # FK_BF16, FK_FP16


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPE_CODES[dtype]


def require_float16ish(name: str, t, ndim: int | None = None, *, dtype=None, strided_rows: bool = False):
    """:func:`require_tensor` for bf16 or fp16 (or the given one of the two). ``strided_rows``
    allows any stride of the first dimension, the others dense."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if (t.dtype not in _DTYPE_CODES) if dtype is None else (t.dtype != dtype):
        raise TypeError(f"{name} must be {'bfloat16 or float16' if dtype is None else dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}")
    if not t.is_contiguous() and not (strided_rows and t.shape[0] > 0 and t[0].is_contiguous()):
        raise ValueError(f"{name} must be {'dense behind its first dimension' if strided_rows else 'contiguous (row-major)'}")
    return t


class launching_on:
    """``with launching_on(dev, stream) as handle``: the library's current device is ``dev``
    inside, and what was current before is current again after, in torch and in the library."""

    __slots__ = ("dev", "stream", "guard", "before")

    def __init__(self, dev: torch.device, stream=None):
        self.dev, self.stream = dev, stream

    def __enter__(self) -> int:
        self.before = torch.cuda.current_device()
        self.guard = None
        if self.dev.index is not None and self.dev.index != self.before:
            self.guard = torch.cuda.device(self.dev)
            self.guard.__enter__()
        return stream_for(self.dev, self.stream)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
            _native.use_device(self.before)
        return False


def scratch(nbytes: int, dev: torch.device, stream_handle: int) -> torch.Tensor:
    """Uninitialised bytes for one call on the given stream. Taken from torch's allocator on that
    stream, so a block is reused only by work behind the call (and, in a captured graph, only by
    that graph)."""
    if stream_handle == torch.cuda.current_stream(dev).cuda_stream:
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream_handle, device=dev)):
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
