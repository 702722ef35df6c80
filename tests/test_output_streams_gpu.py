"""Outputs that the caller leaves to a call on another stream than torch's current one (GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import (
    cache_attention,
    cache_evict,
    flash_attention,
    linear,
    lora_linear,
    pack_w4,
    swiglu_gemm,
    w4_linear,
)

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def check_pending_copy(shape, dtype, call):
    """``call(stream)`` leaves an output of the given shape to the package. A block of that size that the
    current stream has freed, but not read yet, must not become that output."""
    side = torch.cuda.Stream()
    call(side)  # kernels are loaded
    copy = torch.zeros(shape, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    block = torch.full(shape, 7, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)  # some 20 ms
    copy.copy_(block)
    del block
    result = call(side)
    torch.cuda.synchronize()
    assert (copy == 7).all()
    return result


def test_w4_linear():
    q = torch.randint(0, 16, (20000, 256), dtype=torch.uint8, device="cuda")
    w = pack_w4(q, torch.rand(20000, 4, device="cuda").to(BF16))
    x = torch.randn(64, 256, device="cuda").to(BF16)
    want = w4_linear(x, w)
    assert torch.equal(check_pending_copy((64, 20000), BF16, lambda s: w4_linear(x, w, stream=s)), want)


def test_cache_attention():
    B, L, Hkv, G, D = 200, 32, 8, 4, 128
    q = torch.randn(B, Hkv * G, D, device="cuda").to(BF16)
    k = torch.randn(B, L, Hkv, D, device="cuda").to(BF16)
    lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
    want, want_lse = cache_attention(q, k, k, lens)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    got, _ = check_pending_copy((B, Hkv * G, D), BF16, lambda s: cache_attention(q, k, k, lens, None, lse, stream=s))
    assert torch.equal(got, want)
    _, got = check_pending_copy((B, Hkv * G), torch.float32,
                                lambda s: cache_attention(q, k, k, lens, out, None, stream=s))
    assert torch.equal(got, want_lse)


def test_cache_evict():
    B, L, H, D, budget = 64, 64, 8, 64, 1024
    k = torch.randn(B, L, H, D, device="cuda").to(BF16)
    lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
    mass = torch.rand(B, H, L, device="cuda")
    args = (k, k, lens, mass, torch.empty_like(k), torch.empty_like(k), torch.empty_like(lens), torch.empty_like(mass))
    want = cache_evict(*args, budget)
    got = check_pending_copy((B, H, budget), torch.int32, lambda s: cache_evict(*args, budget, stream=s))
    assert torch.equal(got, want)


def test_the_default_stream_named_from_another_one():
    w = pack_w4(torch.randint(0, 16, (200, 256), dtype=torch.uint8, device="cuda"),
                torch.rand(200, 4, device="cuda").to(BF16))
    x = torch.randn(3, 256, device="cuda").to(BF16)
    q, k = torch.randn(3, 8, 128, device="cuda").to(BF16), torch.randn(3, 100, 2, 128, device="cuda").to(BF16)
    lens = torch.tensor([100, 0, 31], dtype=torch.int32, device="cuda")
    want, (out, lse) = w4_linear(x, w), cache_attention(q, k, k, lens)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for stream in (0, torch.cuda.default_stream()):
            y, (o, l) = w4_linear(x, w, stream=stream), cache_attention(q, k, k, lens, stream=stream)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(o, out) and torch.equal(l, lse)


def test_no_rows():
    w = pack_w4(torch.zeros(32, 64, dtype=torch.uint8, device="cuda"), torch.ones(32, 1, device="cuda").to(BF16))
    assert w4_linear(torch.empty(0, 64, dtype=BF16, device="cuda"), w).shape == (0, 32)
    q, k = torch.empty(0, 4, 64, device="cuda").to(BF16), torch.empty(0, 8, 2, 64, device="cuda").to(BF16)
    lens, mass = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 2, 8, device="cuda")
    out, lse = cache_attention(q, k, k, lens, mass=mass)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_linear_family_and_prefill_attention():
    x = torch.randn(64, 256, device="cuda").to(BF16)
    w = (0.05 * torch.randn(20000, 256, device="cuda")).to(BF16)
    a, b = torch.randn(16, 256, device="cuda").to(BF16), torch.randn(20000, 16, device="cuda").to(BF16)
    q = torch.randn(2, 8, 1024, 128, device="cuda").to(BF16)
    k = torch.randn(2, 2, 1024, 128, device="cuda").to(BF16)
    for shape, call in (((64, 20000), lambda s: linear(x, w, stream=s)),
                        ((64, 10000), lambda s: swiglu_gemm(x, w, stream=s)),
                        ((64, 20000), lambda s: lora_linear(x, w, b, lora_a=a, stream=s)),
                        (tuple(q.shape), lambda s: flash_attention(q, k, k, stream=s))):
        want = call(None)
        assert torch.equal(check_pending_copy(shape, BF16, call), want)
    lse_shape = (2, 8, 1024)
    out = torch.empty_like(q)
    want = flash_attention(q, k, k, out, return_lse=True)[1]
    got = check_pending_copy(lse_shape, torch.float32, lambda s: flash_attention(q, k, k, out, return_lse=True, stream=s))
    assert torch.equal(got[1], want)
