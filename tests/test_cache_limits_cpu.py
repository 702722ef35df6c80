"""Sizes past the range of a C int are refused, not truncated."""
import pytest

from fused_kernels_cutedsl_lib_b200 import _native, cache_attention_workspace_bytes


def test_workspace_bytes():
    assert cache_attention_workspace_bytes(1, 1 << 30, 1, 1, 64) > 0
    for tokens in ((1 << 30) + 1, (1 << 31) - 1, 1 << 32, (1 << 32) + 64):
        with pytest.raises(ValueError):
            cache_attention_workspace_bytes(1, tokens, 1, 1, 64)


def test_entry_points_refuse_before_launch():
    lib = _native.load()

    def evict(L=64, lo=32, budget=32):
        return lib.fk_cache_evict(16, 128, None, 16, 16, 1 << 40, 64, 192, None, 48, 32, 1 << 40, 16, 1, L, 0, 0, lo, 0,
                                  0, 2, 256, budget, 0, 0, None)

    for bad in (dict(L=(1 << 31) - 1), dict(lo=(1 << 30) + 1), dict(lo=(1 << 31) - 1, budget=(1 << 31) - 1)):
        assert evict(**bad) == -1, bad
        assert b"2^30" in lib.fk_last_error()
    assert lib.fk_cache_attn_fwd(16, 512, 16, 16, None, 16, None, None, 0, 16, 16, 0, 1, (1 << 31) - 1, 0, 0, 4, 2, 128,
                                 1.0, 16, 1 << 62, None) == -1
    assert b"2^30" in lib.fk_last_error()
