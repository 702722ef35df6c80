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
from ._tensors import (current_device, dtype_code, empty_on, launch_stream, on_device, one_device, require_dense,
                       require_half, require_tensor)

HEAD_DIMS = (64, 128)
MAX_GROUP = 16
MAX_TOKENS = 1 << 30  # of a row, in a cache or to be kept

_HALF = (torch.bfloat16, torch.float16)
_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8


def cache_attention_workspace_bytes(batch: int, max_seqlen: int, num_heads_q: int, num_heads_kv: int,
                                    head_dim: int, mass: bool = False) -> int:
    """Bytes of scratch a :func:`cache_attention` call of these sizes needs on the current device
    (``max_seqlen``: tokens a row of the cache can hold)."""
    n = ctypes.c_size_t(0)
    if max_seqlen > MAX_TOKENS:
        raise ValueError(f"max_seqlen must be <= {MAX_TOKENS}, got {max_seqlen}")
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


def _quick_attention(q, k, v, lens, out, lse, table, mass, mass_out, softmax_scale, workspace):
    """The scale if every argument is as :func:`_check_attention` wants it, by the shortest tests, else
    None. The checks are most of a small call's time: these take 3 us, the others 8."""
    try:
        B, Hq, D = q.shape
        rows, L, Hkv, Dk = k.shape
        dt, idx = q.dtype, q.get_device()
        scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
        if not (dt in _HALF and idx >= 0 and Dk == D and D in HEAD_DIMS and Hkv and Hq % Hkv == 0 and L and rows
                and Hkv <= Hq <= MAX_GROUP * Hkv and q.is_contiguous() and math.isfinite(scale)
                and k.dtype == dt and k.is_contiguous() and k.get_device() == idx
                and v.dtype == dt and v.is_contiguous() and v.get_device() == idx and v.shape == k.shape
                and lens.dtype == _I32 and lens.is_contiguous() and lens.get_device() == idx and lens.shape == (B,)
                and out.dtype == dt and out.is_contiguous() and out.get_device() == idx and out.numel() == q.numel()
                and lse.dtype == _F32 and lse.is_contiguous() and lse.get_device() == idx and lse.shape == (B, Hq)):
            return None
        if table is None:
            if rows != B:
                return None
        else:
            if not (table.dtype == _I32 and table.is_contiguous() and table.get_device() == idx):
                return None
            tb, tp = table.shape
            if tb != B or tp < 1:
                return None
            L *= tp
        if L > MAX_TOKENS:
            return None
        if mass is not None:
            if not (mass.dtype == _F32 and mass.is_contiguous() and mass.get_device() == idx and mass.dim() == 3
                    and mass.shape[0] == B and mass.shape[1] == Hkv and mass.shape[2] >= L):
                return None
            if mass_out is not mass and not (mass_out.dtype == _F32 and mass_out.is_contiguous()
                                             and mass_out.get_device() == idx and mass_out.shape == mass.shape):
                return None
        elif mass_out is not None:
            return None
        if workspace is not None and not (workspace.dtype == _U8 and workspace.is_contiguous()
                                          and workspace.get_device() == idx and workspace.dim() == 1):
            return None
        return scale
    except (AttributeError, TypeError, ValueError):
        return None  # something is no tensor, or has other dimensions: the checks say what


def _check_attention(q, k_cache, v_cache, cache_seqlens, out, lse, block_table, mass, mass_out, softmax_scale,
                     workspace):
    """Raises what is wrong with the arguments of :func:`cache_attention`; the scale."""
    require_half("q", q, strided_rows=True)
    dt = q.dtype
    if q.dim() != 3:
        raise ValueError(f"q must be [B, Hq, D] or [B, 1, Hq, D], got {tuple(q.shape)}")
    B, Hq, D = q.shape
    require_half("k_cache", k_cache, 4, dtype=dt)
    rows, L, Hkv, Dk = k_cache.shape
    require_dense("v_cache", v_cache, dt, k_cache.shape)
    if Dk != D or D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} in q and the caches, got {D} and {Dk}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > MAX_GROUP:
        raise ValueError(f"num_heads_q ({Hq}) must be a multiple of num_heads_kv ({Hkv}), ratio <= {MAX_GROUP}")
    require_dense("cache_seqlens", cache_seqlens, torch.int32, (B,))
    page = pages = 0
    if block_table is not None:
        _check_table("block_table", block_table, B)
        page, pages = L, rows
        L = block_table.shape[1] * page
    elif rows != B:
        raise ValueError(f"the caches hold {rows} rows but q has {B}")
    if L < 1 or (block_table is not None and pages < 1):
        raise ValueError("the cache holds no tokens")
    if L > MAX_TOKENS:
        raise ValueError(f"a row of the cache holds {L} tokens, at most {MAX_TOKENS} are supported")
    cap = 0
    if mass is not None:
        require_tensor("mass", mass, torch.float32, 3)
        cap = mass.shape[2]
        if mass.shape[0] != B or mass.shape[1] != Hkv or cap < L:
            raise ValueError(f"mass must be [{B}, {Hkv}, >= {L}], got {tuple(mass.shape)}")
        if mass_out is not mass:
            require_dense("mass_out", mass_out, torch.float32, (B, Hkv, cap))
    elif mass_out is not None:
        raise ValueError("mass_out needs mass")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale):
        raise ValueError(f"softmax_scale must be finite, got {softmax_scale}")
    if out is not None:
        require_half("out", out, dtype=dt)
        if out.numel() != B * Hq * D:
            raise ValueError(f"out must hold {B}x{Hq}x{D} elements, got shape {tuple(out.shape)}")
    if lse is not None:
        require_dense("lse", lse, torch.float32, (B, Hq))
    if workspace is not None:
        require_tensor("workspace", workspace, torch.uint8, 1)
    one_device(q, k_cache, v_cache, cache_seqlens, block_table, mass, mass_out, out, lse, workspace)
    return scale


def cache_attention(q, k_cache, v_cache, cache_seqlens, out=None, lse=None, *, block_table=None, mass=None,
                    mass_out=None, softmax_scale=None, workspace=None, stream=None):
    """``out = softmax(q K^T * scale) V`` per row over its first ``cache_seqlens[b]`` tokens; returns ``(out, lse)``.

    ``q`` [B, Hq, D] or [B, 1, Hq, D] (rows may be strided, e.g. the q columns of
    a fused QKV output); caches [B, L, Hkv, D], or with ``block_table`` int32
    [B, pages] pools [num_pages, page_size, Hkv, D]. ``mass`` fp32
    [B, Hkv, >= L]: for every token j < len,
    ``mass_out[b, h, j] = mass[b, h, j] + sum over h's q heads of the weight of j``;
    ``mass_out`` defaults to ``mass`` (else: other memory), and entries behind the lengths stay as they
    are. An empty row gives 0 and lse -inf. An ``out``, ``lse`` or ``workspace`` left to the call is memory of the
    stream it runs on (``stream``, or torch's current one).
    """
    if isinstance(q, torch.Tensor) and q.dim() == 4 and q.shape[1] == 1:
        q = q.squeeze(1)
    if mass_out is None:
        mass_out = mass
    scale = None
    if out is not None and lse is not None:
        scale = _quick_attention(q, k_cache, v_cache, cache_seqlens, out, lse, block_table, mass, mass_out,
                                 softmax_scale, workspace)
    if scale is None:
        scale = _check_attention(q, k_cache, v_cache, cache_seqlens, out, lse, block_table, mass, mass_out, softmax_scale,
                                 workspace)
    B, Hq, D = q.shape
    rows, L, Hkv = k_cache.shape[:3]
    idx = q.get_device()
    page = pages = 0
    if block_table is not None:
        page, pages = L, rows
        L = block_table.shape[1] * page
    if idx != current_device():
        with on_device(idx):
            return cache_attention(q, k_cache, v_cache, cache_seqlens, out, lse, block_table=block_table, mass=mass,
                                   mass_out=mass_out, softmax_scale=softmax_scale, workspace=workspace, stream=stream)
    st = launch_stream(idx, stream)
    if out is None:
        out = empty_on((B, Hq, D), q.dtype, idx, st)
    if lse is None:
        lse = empty_on((B, Hq), torch.float32, idx, st)
    if B == 0:
        return out, lse
    if workspace is None:
        workspace = empty_on(cache_attention_workspace_bytes(B, L, Hq, Hkv, D, mass is not None), torch.uint8, idx, st)
    _native.check(_native.load().fk_cache_attn_fwd(
        q.data_ptr(), q.stride(0) if B > 1 else Hq * D, k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr() if block_table is not None else None, cache_seqlens.data_ptr(),
        mass.data_ptr() if mass is not None else None, mass_out.data_ptr() if mass is not None else None,
        mass.shape[2] if mass is not None else 0, out.data_ptr(), lse.data_ptr(), dtype_code(q.dtype), B, L, page,
        pages, Hq, Hkv, D, scale, workspace.data_ptr(), workspace.numel(), st))
    return out, lse


def _meet(a: int, na: int, b: int, nb: int) -> bool:
    """Whether the byte ranges [a, a + na) and [b, b + nb) meet."""
    return a < b + nb and b < a + na


def _overlaps(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, block_table, out_block_table):
    """What of an eviction's outputs meets other memory it must not, or None."""
    pk, pv, pko, pvo = k_cache.data_ptr(), v_cache.data_ptr(), k_out.data_ptr(), v_out.data_ptr()
    nb, nbo = k_cache.numel() * 2, k_out.numel() * 2  # bytes of each input and output cache
    same_pool = (block_table is not None and out_block_table is not None and pko == pk and pvo == pv
                 and block_table.data_ptr() != out_block_table.data_ptr())
    if not same_pool and (_meet(pko, nbo, pk, nb) or _meet(pko, nbo, pv, nb) or _meet(pvo, nbo, pk, nb)
                          or _meet(pvo, nbo, pv, nb)):
        return "the output caches must not overlap the input caches"
    pm, pmo, pl, plo = mass.data_ptr(), mass_out.data_ptr(), cache_seqlens.data_ptr(), seqlens_out.data_ptr()
    if (_meet(pko, nbo, pvo, nbo) or _meet(pm, mass.numel() * 4, pmo, mass_out.numel() * 4)
            or _meet(pl, 4 * cache_seqlens.numel(), plo, 4 * cache_seqlens.numel())):
        return "k_out and v_out, mass and mass_out, and the lengths must not overlap"
    return None


def _quick_evict(k, v, lens, mass, k_out, v_out, lens_out, mass_out, budget, sinks, recent, table, out_table, kept):
    """Whether every argument is as :func:`_check_evict` wants it, by the shortest tests."""
    try:
        rows, L, H, D = k.shape
        rows_out, L_out, h_out, d_out = k_out.shape
        dt, idx = k.dtype, k.get_device()
        (B,) = lens.shape
        if not (dt in _HALF and idx >= 0 and h_out == H and d_out == D and H and D and D % 8 == 0 and L
                and 1 <= budget <= MAX_TOKENS and sinks >= 0 and recent >= 0 and sinks + recent <= budget and k.is_contiguous()
                and v.dtype == dt and v.is_contiguous() and v.get_device() == idx and v.shape == k.shape
                and k_out.dtype == dt and k_out.is_contiguous() and k_out.get_device() == idx
                and v_out.dtype == dt and v_out.is_contiguous() and v_out.get_device() == idx
                and v_out.shape == k_out.shape
                and lens.dtype == _I32 and lens.is_contiguous() and lens.get_device() == idx
                and lens_out.dtype == _I32 and lens_out.is_contiguous() and lens_out.get_device() == idx
                and lens_out.shape == lens.shape
                and mass.dtype == _F32 and mass.is_contiguous() and mass.get_device() == idx
                and mass_out.dtype == _F32 and mass_out.is_contiguous() and mass_out.get_device() == idx
                and kept.dtype == _I32 and kept.is_contiguous() and kept.get_device() == idx
                and kept.shape == (B, H, budget)):
            return False
        for t, n in ((table, rows), (out_table, rows_out)):
            if t is None:
                if n != B:
                    return False
            elif not (t.dtype == _I32 and t.is_contiguous() and t.get_device() == idx and t.dim() == 2
                      and t.shape[0] == B and t.shape[1] >= 1):
                return False
        if table is not None:
            L *= table.shape[1]
        if out_table is not None:
            L_out *= out_table.shape[1]
        need = min(budget, L)
        mb, mh, cap = mass.shape
        ob, oh, out_cap = mass_out.shape
        return (L <= MAX_TOKENS and L_out <= MAX_TOKENS and L_out >= need and mb == B and mh == H and cap >= L and ob == B and oh == H and out_cap >= need
                and _overlaps(k, v, lens, mass, k_out, v_out, lens_out, mass_out, table, out_table) is None)
    except (AttributeError, TypeError, ValueError):
        return False  # something is no tensor, or has other dimensions: the checks say what


def _check_evict(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, budget, sinks, recent,
                 block_table, out_block_table, kept):
    """Raises what is wrong with the arguments of :func:`cache_evict`."""
    require_half("k_cache", k_cache, 4)
    dt = k_cache.dtype
    rows, L, Hkv, D = k_cache.shape
    require_dense("v_cache", v_cache, dt, k_cache.shape)
    require_half("k_out", k_out, 4, dtype=dt)
    rows_out, L_out, h_out, d_out = k_out.shape
    if h_out != Hkv or d_out != D:
        raise ValueError(f"k_out and v_out must be [.., .., {Hkv}, {D}], got {tuple(k_out.shape)}")
    require_dense("v_out", v_out, dt, k_out.shape)
    if Hkv < 1 or D < 8 or D % 8:
        raise ValueError(f"head_dim must be a positive multiple of 8, got {D}")
    require_tensor("cache_seqlens", cache_seqlens, torch.int32, 1)
    B = cache_seqlens.shape[0]
    require_dense("seqlens_out", seqlens_out, torch.int32, (B,))
    if budget < 1 or budget > MAX_TOKENS or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget ({budget}) must lie in [1, {MAX_TOKENS}] and sinks ({sinks}) + recent ({recent}) must lie in "
                         f"[0, budget]")
    page = pages = page_out = pages_out = 0
    if block_table is not None:
        _check_table("block_table", block_table, B)
        page, pages = L, rows
        L = block_table.shape[1] * page
    elif rows != B:
        raise ValueError(f"the caches hold {rows} rows but there are {B} lengths")
    if out_block_table is not None:
        _check_table("out_block_table", out_block_table, B)
        page_out, pages_out = L_out, rows_out
        L_out = out_block_table.shape[1] * page_out
    elif rows_out != B:
        raise ValueError(f"the output caches hold {rows_out} rows but there are {B} lengths")
    need = min(budget, L)
    if max(L, L_out) > MAX_TOKENS:
        raise ValueError(f"rows of the caches hold {L} and {L_out} tokens, at most {MAX_TOKENS} are supported")
    if L < 1 or L_out < need:
        raise ValueError(f"the output cache holds {L_out} tokens per row, needs {need} (and the input at least 1)")
    require_tensor("mass", mass, torch.float32, 3)
    require_tensor("mass_out", mass_out, torch.float32, 3)
    cap, cap_out = mass.shape[2], mass_out.shape[2]
    if mass.shape[0] != B or mass.shape[1] != Hkv or cap < L:
        raise ValueError(f"mass must be [{B}, {Hkv}, >= {L}], got {tuple(mass.shape)}")
    if mass_out.shape[0] != B or mass_out.shape[1] != Hkv or cap_out < need:
        raise ValueError(f"mass_out must be [{B}, {Hkv}, >= {need}], got {tuple(mass_out.shape)}")
    if kept is not None:
        require_dense("kept", kept, torch.int32, (B, Hkv, budget))
    one_device(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, block_table,
               out_block_table, kept)
    wrong = _overlaps(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, block_table,
                      out_block_table)
    if wrong is not None:
        raise ValueError(wrong)


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
    stay as they are. A ``kept`` left to the call is memory of the stream it runs on.

    The output cache is other memory than the input cache, or other pages of the
    same pools: ``out_block_table`` must name no page twice, and none that
    ``block_table`` names for a live token.
    """
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if kept is None or not _quick_evict(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, budget,
                                        sinks, recent, block_table, out_block_table, kept):
        _check_evict(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, budget, sinks, recent,
                     block_table, out_block_table, kept)
    rows, L, Hkv, D = k_cache.shape
    rows_out, L_out = k_out.shape[:2]
    B, idx = cache_seqlens.shape[0], k_cache.get_device()
    page = pages = page_out = pages_out = 0
    if block_table is not None:
        page, pages = L, rows
        L = block_table.shape[1] * page
    if out_block_table is not None:
        page_out, pages_out = L_out, rows_out
        L_out = out_block_table.shape[1] * page_out
    if idx != current_device():
        with on_device(idx):
            return cache_evict(k_cache, v_cache, cache_seqlens, mass, k_out, v_out, seqlens_out, mass_out, budget,
                               sinks=sinks, recent=recent, block_table=block_table, out_block_table=out_block_table,
                               kept=kept, stream=stream)
    st = launch_stream(idx, stream)
    if kept is None:
        kept = empty_on((B, Hkv, budget), torch.int32, idx, st)
    if B == 0:
        return kept
    _native.check(_native.load().fk_cache_evict(
        k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr() if block_table is not None else None,
        cache_seqlens.data_ptr(), mass.data_ptr(), mass.shape[2], k_out.data_ptr(), v_out.data_ptr(),
        out_block_table.data_ptr() if out_block_table is not None else None, seqlens_out.data_ptr(),
        mass_out.data_ptr(), mass_out.shape[2], kept.data_ptr(), B, L,
        page, pages, L_out, page_out, pages_out, Hkv, D * 2, budget, sinks, recent, st))
    return kept
