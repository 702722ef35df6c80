"""Cache attention and eviction: refusals that need no GPU, and the plain eviction the GPU tests go by."""
import ctypes

import pytest
import torch

import cache_reference as ref
from fused_kernels_cutedsl_lib_b200 import _native, cache_attention, cache_attention_workspace_bytes, cache_evict


def test_workspace_bytes():
    a = cache_attention_workspace_bytes(4, 4096, 32, 8, 128)
    b = cache_attention_workspace_bytes(4, 4096, 32, 8, 128, mass=True)
    assert b - a == 4 * 4096 * 32 * 4  # one fp32 score per token and q head
    for bad in ((0, 1, 1, 1, 64), (1, 0, 1, 1, 64), (1, 1, 3, 2, 64), (1, 1, 17, 1, 64), (1, 1, 1, 1, 96)):
        with pytest.raises(ValueError):
            cache_attention_workspace_bytes(*bad)


def test_entry_points_refuse_before_launch():
    lib = _native.load()

    def attn(q=16, stride=512, k=16, table=None, mass=None, mass_out=None, cap=0, dtype=0, b=1, L=64, bs=0, nb=0, hq=4,
             hkv=2, d=128, scale=1.0, ws=16, n=1 << 30):
        return lib.fk_cache_attn_fwd(q, stride, k, 16, table, 16, mass, mass_out, cap, 16, 16, dtype, b, L, bs, nb, hq,
                                     hkv, d, scale, ws, n, None)

    for bad in (dict(q=None), dict(q=18), dict(stride=511), dict(k=24), dict(mass=16), dict(mass=16, mass_out=16, cap=63),
                dict(dtype=3), dict(b=0), dict(L=0), dict(table=16, bs=0, nb=1), dict(table=16, bs=24, nb=1),
                dict(table=16, bs=16, nb=0), dict(hq=5), dict(hq=64), dict(d=80), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(ws=None), dict(ws=8), dict(n=100)):
        assert attn(**bad) == -1, bad
        assert lib.fk_last_error()

    def evict(k=16, ko=64, table=None, otable=None, mass=16, mo=32, cap=64, ocap=32, b=1, L=64, bs=0, nb=0, lo=32,
              obs=0, onb=0, h=2, rb=256, budget=32, sinks=0, recent=0, new=48):
        return lib.fk_cache_evict(k, 128, table, 16, mass, cap, ko, 192, otable, new, mo, ocap, 16, b, L, bs, nb, lo,
                                  obs, onb, h, rb, budget, sinks, recent, None)

    for bad in (dict(k=None), dict(k=20), dict(ko=16), dict(ko=128), dict(mo=16), dict(cap=63), dict(ocap=31), dict(b=0),
                dict(L=0), dict(lo=31), dict(rb=24), dict(rb=0), dict(budget=0), dict(sinks=-1), dict(recent=-1),
                dict(sinks=20, recent=13), dict(new=16), dict(table=16, bs=24, nb=1), dict(table=16, bs=0, nb=1),
                dict(otable=16, obs=24, onb=1), dict(otable=16, obs=16, onb=0), dict(h=0)):
        assert evict(**bad) == -1, bad
        assert lib.fk_last_error()
    n = ctypes.c_size_t(0)
    assert lib.fk_cache_attn_workspace_bytes(1, 1, 1, 1, 64, 0, None) == -1
    assert lib.fk_cache_attn_workspace_bytes(1, 1, 1, 1, 64, 0, ctypes.byref(n)) == 0 and n.value > 0


def test_python_entry_points_refuse_cpu_tensors():
    q, k = torch.zeros(1, 4, 64, dtype=torch.float16), torch.zeros(1, 8, 2, 64, dtype=torch.float16)
    lens, mass = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 8)
    with pytest.raises(ValueError):
        cache_attention(q, k, k, lens)
    with pytest.raises(ValueError):
        cache_evict(k, k, lens, mass, k, k, lens, mass, 4)


def test_plain_eviction_by_hand():
    k = torch.zeros(2, 8, 1, 8)
    mass = torch.tensor([[[9., 1, 5, 5, 0, 5, 0, 0]], [[0., 0, 3, 0, 0, 0, 0, 0]]])
    kept, new = ref.evict(k, k, torch.tensor([8, 3]), mass, 4, 1, 1)
    assert kept.tolist() == [[[0, 2, 3, 7]], [[0, 1, 2, -1]]] and new.tolist() == [4, 3]
