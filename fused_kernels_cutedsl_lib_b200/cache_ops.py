"""Attention over a KV cache that keeps count of its tokens, and eviction by that count
(host side of ``csrc/cache_attn.cu`` and ``csrc/cache_evict.cu``).

* :func:`cache_attention`: softmax attention of one new token per sequence over
  a contiguous or paged cache (pages of any size, bf16 or fp16, head_dim 64 or
  128, up to 16 query heads per kv head), which can also add each cached token's
  attention weight to its running sum, its *mass*;
* :func:`cache_evict`: sequences longer than a budget lose the tokens of least
  mass, per kv head; what stays is written to a smaller cache.

Stands beside :func:`~fused_kernels_cutedsl_lib_b200.decoding_attention.decode_attention`
(the softmax form of the reference's ``DAttn1``,
python/cutedsl_kernels/decoding_attention/attn1.py:89-141; semantics of
attn/attempt6_epi_pipeline/attn.py:778-784), which is bf16 with head_dim 128
and pages of a multiple of 64 tokens, and has no masses. A decode loop with a
bounded cache appends (``layer.kv_append``), attends with ``mass=``, and evicts
whenever the cache is full.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native
from ._tensors import (dtype_code, launching_on, ptr, require_float16ish, require_shape, require_tensor, same_device,
                       scratch)

HEAD_DIMS = (64, 128)
MAX_GROUP = 16


def cache_attention_workspace_bytes(batch: int, max_seqlen: int, num_heads_q: int, num_heads_kv: int,
                                    head_dim: int, mass: bool = False) -> int:
    """Bytes of scratch a :func:`cache_attention` call of these sizes needs on the current device
    (``max_seqlen``: tokens a row of the cache can hold)."""
    n = ctypes.c_size_t(0)
    _native.check(_native.load().fk_cache_attn_workspace_bytes(
        int(batch), int(max_seqlen), int(num_heads_q), int(num_heads_kv), int(head_dim), int(bool(mass)),
        ctypes.byref(n)))
    return int(n.value)


def alloc_cache_attention_workspace(batch: int, max_seqlen: int, num_heads_q: int, num_heads_kv: int,
                                    head_dim: int, mass: bool = False, device="cuda") -> torch.Tensor:
    """Scratch for :func:`cache_attention`, of any contents. Calls that may overlap on the GPU
    (other streams, other captured graphs) need one each."""
    dev = torch.device(device)
    with torch.cuda.device(dev):
        n = cache_attention_workspace_bytes(batch, max_seqlen, num_heads_q, num_heads_kv, head_dim, mass)
        return torch.empty(n, dtype=torch.uint8, device=dev)


def _check_table(name, table, batch):
    require_tensor(name, table, torch.int32, 2)
    if table.shape[0] != batch or table.shape[1] < 1:
        raise ValueError(f"{name} must be [{batch}, pages per row], got {tuple(table.shape)}")


def cache_attention(q, k_cache, v_cache, cache_seqlens, out=None, lse=None, *, block_table=None, mass=None,
                    mass_out=None, softmax_scale=None, workspace=None, stream=None):
    """``out = softmax(q K^T * scale) V`` per row over its first ``cache_seqlens[b]`` tokens; returns ``(out, lse)``.

    ``q`` [B, Hq, D] or [B, 1, Hq, D] (rows may be strided, e.g. the q columns of
    a fused QKV output); caches [B, L, Hkv, D], or with ``block_table`` int32
    [B, pages] pools [num_pages, page_size, Hkv, D]. ``mass`` fp32
    [B, Hkv, >= L]: for every token j < len,
    ``mass_out[b, h, j] = mass[b, h, j] + sum over h's q heads of the weight of j``;
    ``mass_out`` defaults to ``mass``, and entries behind the lengths stay as they
    are. An empty row gives 0 and lse -inf.
    """
    require_float16ish("q", q, strided_rows=True)
    dt = q.dtype
    if q.dim() == 4 and q.shape[1] == 1:
        q = q.squeeze(1)
    if q.dim() != 3:
        raise ValueError(f"q must be [B, Hq, D] or [B, 1, Hq, D], got {tuple(q.shape)}")
    B, Hq, D = q.shape
    require_float16ish("k_cache", k_cache, 4, dtype=dt)
    require_float16ish("v_cache", v_cache, 4, dtype=dt)
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must have the same shape, got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    require_tensor("cache_seqlens", cache_seqlens, torch.int32, 1)
    rows, L, Hkv = k_cache.shape[:3]
    if k_cache.shape[3] != D or D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} in q and the caches, got {D} and {k_cache.shape[3]}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > MAX_GROUP:
        raise ValueError(f"num_heads_q ({Hq}) must be a multiple of num_heads_kv ({Hkv}), ratio <= {MAX_GROUP}")
    require_shape("cache_seqlens", cache_seqlens, (B,))
    tensors = [q, k_cache, v_cache, cache_seqlens]
    page = pages = 0
    if block_table is not None:
        _check_table("block_table", block_table, B)
        tensors.append(block_table)
        page, pages = L, rows
        L = block_table.shape[1] * page
    elif rows != B:
        raise ValueError(f"the caches hold {rows} rows but q has {B}")
    if L < 1 or (block_table is not None and pages < 1):
        raise ValueError("the cache holds no tokens")
    if mass is None and mass_out is not None:
        raise ValueError("mass_out needs mass")
    cap = 0
    if mass is not None:
        mass_out = mass if mass_out is None else mass_out
        require_tensor("mass", mass, torch.float32, 3)
        require_tensor("mass_out", mass_out, torch.float32, 3)
        if tuple(mass.shape[:2]) != (B, Hkv) or mass.shape[2] < L or mass_out.shape != mass.shape:
            raise ValueError(f"mass and mass_out must be [{B}, {Hkv}, >= {L}] alike, got {tuple(mass.shape)} and "
                             f"{tuple(mass_out.shape)}")
        cap = mass.shape[2]
        tensors += [mass, mass_out]
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale):
        raise ValueError(f"softmax_scale must be finite, got {softmax_scale}")
    if out is None:
        out = torch.empty((B, Hq, D), dtype=dt, device=q.device)
    else:
        require_tensor("out", out, dt)
        if out.numel() != B * Hq * D:
            raise ValueError(f"out must hold {B}x{Hq}x{D} elements, got shape {tuple(out.shape)}")
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device)
    else:
        require_tensor("lse", lse, torch.float32, 2)
        require_shape("lse", lse, (B, Hq))
    tensors += [out, lse]
    if workspace is not None:
        require_tensor("workspace", workspace, torch.uint8, 1)
        tensors.append(workspace)
    dev = same_device(*tensors)
    if B == 0:
        return out, lse
    with launching_on(dev, stream) as st:
        if workspace is None:
            workspace = scratch(cache_attention_workspace_bytes(B, L, Hq, Hkv, D, mass is not None), dev, st)
        _native.check(_native.load().fk_cache_attn_fwd(
            ptr(q), q.stride(0) if B > 1 else Hq * D, ptr(k_cache), ptr(v_cache),
            ptr(block_table) if block_table is not None else None, ptr(cache_seqlens),
            ptr(mass) if mass is not None else None, ptr(mass_out) if mass is not None else None, cap, ptr(out),
            ptr(lse), dtype_code(dt), B, L, page, pages, Hq, Hkv, D, scale, ptr(workspace), workspace.numel(), st))
    return out, lse


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 < b0 + b.numel() * b.element_size() and b0 < a0 + a.numel() * a.element_size()


def cache_evict(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, budget: int, *,
                sinks: int = 0, recent: int = 0, block_table=None, out_block_table=None, kept=None, stream=None):
    """Keep at most ``budget`` tokens of every sequence, those of greatest mass; returns ``kept``.

    Per row longer than ``budget`` and per kv head: the first ``sinks`` tokens, the
    last ``recent`` and the ``budget - sinks - recent`` others of greatest
    ``mass`` [B, Hkv, >= L] (equal masses: the earlier token) stay, in order; shorter
    rows stay whole. Their K/V rows go to slots 0.. of ``k_out`` / ``v_out``
    (contiguous [B, L_out, Hkv, D], or pools with ``out_block_table``), their masses
    to ``mass_out`` [B, Hkv, >= min(budget, L)], which is zeroed behind them, the
    lengths to ``seqlens_out`` [B], and the old positions to ``kept`` int32
    [B, Hkv, budget] (-1 behind). Slots of ``k_out`` / ``v_out`` behind the lengths
    stay as they are.

    The output cache is other memory than the input cache, or other pages of the
    same pools: ``out_block_table`` must name no page twice, and none that
    ``block_table`` names for a live token.
    """
    require_float16ish("k_cache", k_cache, 4)
    dt = k_cache.dtype
    require_float16ish("v_cache", v_cache, 4, dtype=dt)
    require_float16ish("k_out", k_out, 4, dtype=dt)
    require_float16ish("v_out", v_out, 4, dtype=dt)
    if k_cache.shape != v_cache.shape or k_out.shape != v_out.shape:
        raise ValueError("K and V caches must have the same shapes")
    require_tensor("cache_seqlens", cache_seqlens, torch.int32, 1)
    require_tensor("seqlens_out", seqlens_out, torch.int32, 1)
    require_tensor("mass", mass, torch.float32, 3)
    require_tensor("mass_out", mass_out, torch.float32, 3)
    rows, L, Hkv, D = k_cache.shape
    rows_out, L_out = k_out.shape[:2]
    B = cache_seqlens.shape[0]
    if tuple(k_out.shape[2:]) != (Hkv, D):
        raise ValueError(f"k_out and v_out must be [.., .., {Hkv}, {D}], got {tuple(k_out.shape)}")
    if Hkv < 1 or D < 8 or D % 8:
        raise ValueError(f"head_dim must be a positive multiple of 8, got {D}")
    require_shape("seqlens_out", seqlens_out, (B,))
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget ({budget}) must be >= 1 and sinks ({sinks}) + recent ({recent}) must lie in "
                         f"[0, budget]")
    tensors = [k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out]
    page = pages = page_out = pages_out = 0
    if block_table is not None:
        _check_table("block_table", block_table, B)
        tensors.append(block_table)
        page, pages = L, rows
        L = block_table.shape[1] * page
    elif rows != B:
        raise ValueError(f"the caches hold {rows} rows but there are {B} lengths")
    if out_block_table is not None:
        _check_table("out_block_table", out_block_table, B)
        tensors.append(out_block_table)
        page_out, pages_out = L_out, rows_out
        L_out = out_block_table.shape[1] * page_out
    elif rows_out != B:
        raise ValueError(f"the output caches hold {rows_out} rows but there are {B} lengths")
    need = min(budget, L)
    if L < 1 or L_out < need:
        raise ValueError(f"the output cache holds {L_out} tokens per row, needs {need} (and the input at least 1)")
    if tuple(mass.shape[:2]) != (B, Hkv) or mass.shape[2] < L:
        raise ValueError(f"mass must be [{B}, {Hkv}, >= {L}], got {tuple(mass.shape)}")
    if tuple(mass_out.shape[:2]) != (B, Hkv) or mass_out.shape[2] < need:
        raise ValueError(f"mass_out must be [{B}, {Hkv}, >= {need}], got {tuple(mass_out.shape)}")
    if kept is None:
        kept = torch.empty((B, Hkv, budget), dtype=torch.int32, device=k_cache.device)
    else:
        require_tensor("kept", kept, torch.int32, 3)
        require_shape("kept", kept, (B, Hkv, budget))
    tensors.append(kept)
    dev = same_device(*tensors)
    same_pool = (block_table is not None and out_block_table is not None and not _overlap(block_table, out_block_table)
                 and k_out.data_ptr() == k_cache.data_ptr() and v_out.data_ptr() == v_cache.data_ptr())
    if not same_pool and any(_overlap(a, b) for a in (k_out, v_out) for b in (k_cache, v_cache)):
        raise ValueError("the output caches must not overlap the input caches")
    if _overlap(k_out, v_out) or _overlap(mass, mass_out) or _overlap(cache_seqlens, seqlens_out):
        raise ValueError("k_out and v_out, mass and mass_out, and the lengths must not overlap")
    if B == 0:
        return kept
    with launching_on(dev, stream) as st:
        _native.check(_native.load().fk_cache_evict(
            ptr(k_cache), ptr(v_cache), ptr(block_table) if block_table is not None else None, ptr(cache_seqlens),
            ptr(mass), mass.shape[2], ptr(k_out), ptr(v_out),
            ptr(out_block_table) if out_block_table is not None else None, ptr(seqlens_out), ptr(mass_out),
            mass_out.shape[2], ptr(kept), B, L, page, pages, L_out, page_out, pages_out, Hkv, D * k_cache.element_size(),
            budget, sinks, recent, st))
    return kept
