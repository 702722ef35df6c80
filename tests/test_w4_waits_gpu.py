"""The 4-bit linear's bounded waits (GPU)."""
import ctypes

import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import _native, pack_w4, w4_linear

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def make(m, n, k, group):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    q = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    s = (0.004 + 0.008 * torch.rand(n, k // group, generator=g, device="cuda")).to(BF16)
    return torch.randn(m, k, generator=g, device="cuda").to(BF16), pack_w4(q, s)


@pytest.fixture
def wait_limit():
    """Sets the bound of every wait; the built-in one comes back at the end."""
    lib = _native.load()
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    yield lambda ns: _native.check(lib.fk_set_wait_limit_ns(ns))
    _native.check(lib.fk_set_wait_limit_ns(0))


@pytest.mark.parametrize("m,n,k,group", [(1, 512, 8192, 128), (5, 4096, 4096, 32), (16, 40, 20480, 64),
                                         (16, 28672, 1024, 128), (64, 512, 8192, 64), (40, 1000, 4096, 32),
                                         (100, 256, 14336, 128)])
def test_a_long_predecessor_is_waited_for(m, n, k, group, wait_limit):
    """Kernels before the call on its stream that let it start early and then take longer than a wait may:
    three stage barriers whose flags nobody sets, each of which gives up at the bound."""
    lib = _native.load()
    x, w = make(m, n, k, group)
    want = w4_linear(x, w)
    flags, counter, peer = (torch.zeros(8, dtype=torch.int32, device="cuda") for _ in range(3))
    pointers = (ctypes.c_void_p * 2)(flags.data_ptr(), peer.data_ptr())
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    wait_limit(3_000_000)  # 3 ms
    st = torch.cuda.current_stream().cuda_stream
    for _ in range(3):
        _native.check(lib.fk_peer_barrier(counter.data_ptr(), flags.data_ptr(), pointers, 0, 2, st))
    w4_linear(x, w, out)
    torch.cuda.synchronize()
    assert _native.device_error() == 4  # the barriers': a flag's wait ran out
    assert torch.equal(out, want)
    assert int(counter[0]) == 3


# One to eight CTAs per cluster, rows in one and in several rounds, one and two accumulator buffers.
@pytest.mark.parametrize("slab", [0, 1, 9])
@pytest.mark.parametrize("m,n,k,group", [(1, 512, 256, 128), (5, 4096, 4096, 32), (2, 512, 20480, 128),
                                         (16, 28672, 4096, 128), (8, 70000, 800, 32), (16, 40, 20480, 64),
                                         (64, 512, 8192, 64), (40, 1000, 4096, 32), (64, 4096, 14336, 128),
                                         (100, 256, 256, 64)])
def test_a_missing_slab_ends_the_call(m, n, k, group, slab, wait_limit):
    """The first CTA never gets one of its slabs (or all of them, where it has fewer): its warps and those of
    its cluster give up one after the other, the launch completes with the error word set, and
    the next calls are right."""
    lib = _native.load()
    x, w = make(m, n, k, group)
    want = w4_linear(x, w)
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    wait_limit(1_000_000)  # 1 ms
    try:
        _native.check(lib.fk_debug_w4_withhold_slab(slab))
        w4_linear(x, w, out)
        torch.cuda.synchronize()
    finally:
        _native.check(lib.fk_debug_w4_withhold_slab(-1))
    code = _native.device_error()
    if code == 0:  # the CTA has no such slab
        assert slab > 0 and torch.equal(out, want)
    else:
        assert code in (1, 2, 3, 4)
    for _ in range(3):
        w4_linear(x, w, out)
        assert torch.equal(out, want)
    assert _native.device_error() == 0
