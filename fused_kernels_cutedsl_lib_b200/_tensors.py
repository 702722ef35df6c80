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


def raw_current_stream(idx: int) -> int:
    """Torch's current stream on device ``idx`` as an int, without building a Stream object
    (0.1 instead of 2.2 us of host time per call)."""
    return torch._C._cuda_getCurrentRawStream(idx)


if not hasattr(torch._C, "_cuda_getCurrentRawStream"):  # a torch without that accessor
    def raw_current_stream(idx: int) -> int:  # noqa: F811
        return torch.cuda.current_stream(idx).cuda_stream


def stream_for(dev: torch.device, stream=None) -> int:
    """cudaStream_t (as int) to launch on: explicit, else torch's current stream."""
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    _native.use_device(idx)
    if stream is None:
        return raw_current_stream(idx)
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


_DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1}  # FK_BF16, FK_FP16


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPE_CODES[dtype]


def require_half(name: str, t, ndim: int | None = None, *, dtype=None, strided_rows: bool = False) -> None:
    """:func:`require_tensor` for bf16 or fp16 (or the given one of the two). ``strided_rows``
    allows any stride of the first dimension, the others dense."""
    if (isinstance(t, torch.Tensor) and (t.dtype in _DTYPE_CODES if dtype is None else t.dtype == dtype)
            and (ndim is None or t.dim() == ndim) and t.is_cuda
            and (t.is_contiguous() or (strided_rows and t.shape[0] > 0 and t[0].is_contiguous()))):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if (t.dtype not in _DTYPE_CODES) if dtype is None else (t.dtype != dtype):
        raise TypeError(f"{name} must be {'bfloat16 or float16' if dtype is None else dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}")
    raise ValueError(f"{name} must be {'dense behind its first dimension' if strided_rows else 'contiguous (row-major)'}")


def require_dense(name: str, t, dtype: torch.dtype, shape: tuple) -> None:
    """A contiguous CUDA tensor of the given type and shape: :func:`require_tensor` and
    :func:`require_shape` with one pass of checks where nothing is wrong."""
    if (isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape and t.is_cuda and t.is_contiguous()):
        return
    require_tensor(name, t, dtype, len(shape))
    require_shape(name, t, shape)


def one_device(*ts) -> int:
    """Index of the CUDA device that holds every tensor (None entries are passed over)."""
    idx = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != idx:
            same_device(*[u for u in ts if u is not None])
    return idx


# Without torch's test for initialisation: the callers hold a CUDA tensor.
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class on_device:
    """``with on_device(idx)``: device ``idx`` is current in torch; behind it the one that was
    current before is so again, in torch and in the library."""

    def __init__(self, idx: int):
        self.guard, self.before = torch.cuda.device(idx), torch.cuda.current_device()

    def __enter__(self):
        self.guard.__enter__()

    def __exit__(self, *exc):
        self.guard.__exit__(*exc)
        _native.use_device(self.before)


def launch_stream(idx: int, stream=None) -> int:
    """cudaStream_t (as int) to launch on, on the current device ``idx``: explicit, else torch's current."""
    _native.use_device(idx)
    if stream is None:
        return raw_current_stream(idx)
    return stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else int(stream)


def empty_on(shape, dtype: torch.dtype, idx: int, stream_handle: int) -> torch.Tensor:
    """Uninitialised memory for a call on the given stream: scratch, or an output that the caller left to the
    call. Taken from torch's allocator on that stream, so a block is reused only by work behind the call (and, in
    a captured graph, only by that graph), and pending work of another stream never still needs it."""
    dev = torch.device("cuda", idx)
    if stream_handle == raw_current_stream(idx):
        return torch.empty(shape, dtype=dtype, device=dev)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream_handle, device=dev)):
        return torch.empty(shape, dtype=dtype, device=dev)


def result_on(shape, dtype: torch.dtype, dev: torch.device, stream=None) -> torch.Tensor:
    """:func:`empty_on` for a call on ``dev`` with the given ``stream`` argument (None: torch's current one)."""
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if stream is None:
        handle = raw_current_stream(idx)
    else:
        handle = stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else int(stream)
    return empty_on(shape, dtype, idx, handle)
