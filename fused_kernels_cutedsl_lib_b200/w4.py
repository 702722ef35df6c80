"""Linear layer with 4-bit weights and group scales (host side of ``csrc/w4_linear.cu``, ``csrc/w4_tc.cu``).

``y = x @ W.t() (+ residual)`` for the few tokens of a decode step, with
``W[n, k] = (q[n, k] - z[n, k // g]) * s[n, k // g]``, codes ``q`` and zero points
``z`` in [0, 15] and one scale per row and group of ``g`` input features. Stands
beside :func:`~fused_kernels_cutedsl_lib_b200.gemm.skinny_gemm` (``Gemm4SM90``'s
``c = a @ b.t()``, python/cutedsl_kernels/gemm/kernel/attempt4.py:133-168) with a
quarter of its weight bytes; the reference itself has 16-bit weights only.

A weight is laid out once, :func:`pack_w4` (from codes, scales and zero points)
or :func:`quantize_w4` (from a 16- or 32-bit weight), and used any number of times.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native
from ._tensors import (current_device, dtype_code, empty_on, launch_stream, on_device, one_device, require_dense,
                       require_half, same_device)

GROUP_SIZES = (32, 64, 128)
_BLOCK_K = 128  # inputs per block
_SLAB = 2       # input blocks per slab


@dataclass(frozen=True)
class W4Weight:
    """A packed 4-bit weight [N, K]; build it with :func:`pack_w4` or :func:`quantize_w4`."""

    packed: torch.Tensor  # int32, ceil(N/16) * ceil(K/128) blocks of 256 + 2048 / group_size: codes and scales
    n: int
    k: int
    group_size: int
    dtype: torch.dtype    # of the scales, the activations and the output

    def __post_init__(self):
        # The kernels take the sizes on trust: a buffer that is shorter would be read past its end.
        if not isinstance(self.packed, torch.Tensor) or self.packed.dtype != torch.int32:
            raise TypeError("packed must be an int32 tensor")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"dtype must be bfloat16 or float16, got {self.dtype}")
        if self.group_size not in GROUP_SIZES or self.n < 1 or self.k < 1 or self.k % self.group_size:
            raise ValueError(f"group size must be one of {GROUP_SIZES} and divide K, got {self.group_size} for "
                             f"[{self.n}, {self.k}]")
        words = -(-self.n // 16) * -(-self.k // _BLOCK_K) * (256 + 2048 // self.group_size)
        if not self.packed.is_contiguous() or self.packed.numel() != words:
            raise ValueError(f"packed must hold {words} contiguous words for [{self.n}, {self.k}] and groups of "
                             f"{self.group_size}, got shape {tuple(self.packed.shape)}")

    def nbytes(self) -> int:
        return self.packed.numel() * 4

    def dequantize(self) -> torch.Tensor:
        """The weight as fp32 [N, K] (``(q - z) * s``, exact)."""
        nb, kb, words = -(-self.n // 16), -(-self.k // _BLOCK_K), 256 + 2048 // self.group_size
        full = kb // _SLAB
        head = self.packed[:full * _SLAB * nb * words].view(full, nb, _SLAB, words).transpose(0, 1)
        tail = self.packed[full * _SLAB * nb * words:].view(nb, -1, words)
        blocks = torch.cat([head.reshape(nb, -1, words), tail], 1)
        shifts = torch.arange(0, 32, 4, device=self.packed.device, dtype=torch.int32)
        words = _rotate_left(blocks[..., :256], 30)
        q = (words.unsqueeze(-1) >> shifts) & 15
        q = q.view(nb, kb, 2, 8, 4, 4, 2, 4).permute(0, 2, 3, 1, 5, 4, 7, 6)  # [nb, half, g, kb, j, c, pair, odd]
        q = q.reshape(nb * 16, kb * _BLOCK_K)[:self.n, :self.k].float()
        sz = blocks[..., 256:].reshape(nb, -1, 16).transpose(1, 2).reshape(nb * 16, -1)
        sz = sz[:self.n, :self.k // self.group_size]
        both = sz.reshape(-1).contiguous().view(self.dtype).view(self.n, -1, 2).float()
        s, z = both[..., 0], both[..., 1]
        rep = lambda t: t.repeat_interleave(self.group_size, dim=1)  # noqa: E731
        return (q - rep(z)) * rep(s)


def _rotate_left(words: torch.Tensor, n: int) -> torch.Tensor:
    """int32 words rotated by n bits (the shift right of a negative int32 is arithmetic: masked)."""
    return (words << n) | ((words >> (32 - n)) & ((1 << n) - 1))


def pack_w4(q: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> W4Weight:
    """Lay out a 4-bit weight for :func:`w4_linear`.

    ``q`` uint8 [N, K] holds one code (0..15) per element, ``scales`` [N, K // g]
    bf16 or fp16 with g in {32, 64, 128}, ``zeros`` uint8 of the same shape (0..15;
    None: 8 everywhere). Works on any device, and waits for it: the result may be
    used on any stream.
    """
    if not isinstance(q, torch.Tensor) or q.dtype != torch.uint8:
        raise TypeError("q must be a uint8 tensor")
    if not isinstance(scales, torch.Tensor) or scales.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("scales must be a bfloat16 or float16 tensor")
    if q.dim() != 2 or q.shape[0] < 1 or q.shape[1] < 1:
        raise ValueError(f"q must be [N, K], got {tuple(q.shape)}")
    n, k = q.shape
    if scales.dim() != 2 or scales.shape[0] != n or scales.shape[1] < 1 or k % scales.shape[1]:
        raise ValueError(f"scales must be [N={n}, K / group_size], got {tuple(scales.shape)}")
    group = k // scales.shape[1]
    if group not in GROUP_SIZES:
        raise ValueError(f"group size must be one of {GROUP_SIZES}, got {group}")
    if zeros is not None:
        if not isinstance(zeros, torch.Tensor) or zeros.dtype != torch.uint8:
            raise TypeError("zeros must be a uint8 tensor")
        if zeros.shape != scales.shape:
            raise ValueError(f"zeros must have shape {tuple(scales.shape)}, got {tuple(zeros.shape)}")
    same_device(*[t for t in (q, scales, zeros) if t is not None])
    if bool((q > 15).any()) or (zeros is not None and bool((zeros > 15).any())):
        raise ValueError("codes and zero points must lie in [0, 15]")
    dev = q.device
    nb, kb = -(-n // 16), -(-k // _BLOCK_K)
    words = 256 + 2048 // group
    packed = torch.empty(nb, kb, words, dtype=torch.int32, device=dev)
    shifts = torch.arange(0, 32, 4, device=dev, dtype=torch.int32)
    step = max(1, (1 << 25) // (kb * _BLOCK_K * 16))  # row blocks at a time: the int32 codes are 8 times the result
    for b0 in range(0, nb, step):
        rows = q[b0 * 16:(b0 + step) * 16]
        pad = torch.zeros(-(-rows.shape[0] // 16) * 16, kb * _BLOCK_K, dtype=torch.int32, device=dev)
        pad[:rows.shape[0], :k] = rows
        # [nb, half, g, kb, j, c, pair, odd] -> [nb, kb, half, (g, c), j], nibble 4 * odd + pair of the word
        v = pad.view(-1, 2, 8, kb, 4, 4, 4, 2).permute(0, 3, 1, 2, 5, 4, 7, 6).flatten(-2) << shifts
        packed[b0:b0 + v.shape[0], :, :256] = _rotate_left(v.sum(-1, dtype=torch.int32), 2).reshape(-1, kb, 256)
    z = torch.full_like(scales, 8.0) if zeros is None else zeros.to(scales.dtype)
    sz = torch.zeros(nb * 16, kb * _BLOCK_K // group, 2, dtype=scales.dtype, device=dev)
    sz[:n, :k // group, 0] = scales
    sz[:n, :k // group, 1] = z
    packed[..., 256:] = sz.view(torch.int32).view(nb, 16, kb, -1).permute(0, 2, 3, 1).reshape(nb, kb, -1)
    full = kb // _SLAB
    packed = torch.cat([packed[:, :full * _SLAB].view(nb, full, _SLAB, words).transpose(0, 1).reshape(-1),
                        packed[:, full * _SLAB:].reshape(-1)])
    if packed.is_cuda:  # the linear's first copies of a weight do not wait for the kernel before it on the stream
        torch.cuda.current_stream(dev).synchronize()
    return W4Weight(packed, n, k, group, scales.dtype)


def quantize_w4(w: torch.Tensor, group_size: int = 128, symmetric: bool = False, dtype=None) -> W4Weight:
    """Round a weight [N, K] to 4 bits per element with a scale per row and ``group_size`` inputs.

    Asymmetric: the codes span the group's [min(w, 0), max(w, 0)], with a zero point.
    ``symmetric``: scale ``max |w| / 7``, zero point 8. ``dtype`` (default: the
    weight's, bf16 for fp32 weights) is the type of the scales and of the activations.
    Weights that are not finite, or whose scales are not in that type, are refused.
    """
    if not isinstance(w, torch.Tensor) or w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("w must be a bfloat16, float16 or float32 tensor")
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"w must be [N, K], got {tuple(w.shape)}")
    if group_size not in GROUP_SIZES or w.shape[1] % group_size:
        raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide K={w.shape[1]}, got {group_size}")
    dt = dtype if dtype is not None else (torch.bfloat16 if w.dtype == torch.float32 else w.dtype)
    v = w.float().view(w.shape[0], -1, group_size)
    if symmetric:
        scales = (v.abs().amax(-1) / 7.0).to(dt)
        zeros = None
        z = 8.0
    else:
        lo, hi = v.amin(-1).clamp_max(0.0), v.amax(-1).clamp_min(0.0)
        scales = ((hi - lo) / 15.0).to(dt)
        sf = scales.float()
        zeros = torch.where(sf > 0, (-lo / torch.where(sf > 0, sf, 1.0)).round().clamp_(0, 15), 0.0).to(torch.uint8)
        z = zeros.float()[..., None]
    if not bool(torch.isfinite(scales).all()):  # of a NaN or infinite weight as well
        raise ValueError(f"w has an element that is not finite, or whose scale is not finite in {dt}")
    sf = scales.float()[..., None]
    q = torch.where(sf > 0, (v / torch.where(sf > 0, sf, 1.0) + z).round().clamp_(0, 15), z if zeros is not None else 8.0)
    return pack_w4(q.to(torch.uint8).view(w.shape), scales, zeros)


def w4_linear(x, weight: W4Weight, out=None, *, residual=None, stream=None):
    """``out = x @ W.t() (+ residual)`` for a 4-bit weight; returns ``out``.

    ``x`` [M, K] in the weight's dtype, any M (made for decode batches: up to 64
    tokens share one pass over the weight, 32 with groups of 32), rows may be strided (a multiple of 8
    elements); ``out`` and ``residual`` [M, N] dense, ``residual`` may be ``out``.
    Otherwise ``out`` shares no memory with ``x``, ``residual`` or the weight. An ``out`` left to the call
    is memory of the stream it runs on (``stream``, or torch's current one).
    """
    if not isinstance(weight, W4Weight):
        raise TypeError(f"weight must be a W4Weight (pack_w4, quantize_w4), got {type(weight).__name__}")
    n, k, dt = weight.n, weight.k, weight.dtype
    packed = weight.packed
    idx = packed.get_device()
    # The shortest tests first: nothing more to ask if all of them hold.
    if not (isinstance(x, torch.Tensor) and x.dtype == dt and x.dim() == 2 and x.shape[1] == k and x.get_device() == idx
            and idx >= 0 and x.is_contiguous() and k % 8 == 0 and isinstance(out, torch.Tensor)
            and out.dtype == dt and out.get_device() == idx and out.is_contiguous() and out.shape == (x.shape[0], n)
            and (residual is None or (isinstance(residual, torch.Tensor) and residual.dtype == dt
                                      and residual.get_device() == idx and residual.is_contiguous()
                                      and residual.shape == out.shape))):
        require_half("x", x, 2, dtype=dt, strided_rows=True)
        m, xk = x.shape
        if xk != k:
            raise ValueError(f"x is [M, K={xk}] but the weight is [N={n}, K={k}]")
        if m > 1 and (x.stride(0) < k or x.stride(0) % 8):
            raise ValueError(f"x row stride must be >= K and a multiple of 8 elements, got {x.stride(0)}")
        if out is not None:
            require_dense("out", out, dt, (m, n))
        if residual is not None:
            require_dense("residual", residual, dt, (m, n))
        idx = one_device(x, packed, out, residual)
    m = x.shape[0]
    ldx = x.stride(0) if m > 1 else k
    if idx != current_device():
        with on_device(idx):
            return w4_linear(x, weight, out, residual=residual, stream=stream)
    st = launch_stream(idx, stream)
    if out is None:
        out = empty_on((m, n), dt, idx, st)
    if m == 0:
        return out
    _native.check(_native.load().fk_w4_linear(
        x.data_ptr(), ldx, packed.data_ptr(),
        residual.data_ptr() if residual is not None else None, out.data_ptr(), dtype_code(dt), m, n, k,
        weight.group_size, st))
    return out
