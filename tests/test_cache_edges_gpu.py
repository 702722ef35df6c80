"""Corners of the cache operators: non-finite keys and values, weights far apart, sizes past an int (GPU)."""
import math

import pytest
import torch

import cache_reference as ref
from fused_kernels_cutedsl_lib_b200 import _native, cache_attention, cache_evict

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def make(B, L, Hkv, G, D, dtype, lens, seed=0):
    """q, caches with NaN behind every length, lengths and masses."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (1.5 * torch.randn(B, Hkv * G, D, generator=g, device="cuda")).to(dtype)
    k = torch.randn(B, L, Hkv, D, generator=g, device="cuda").to(dtype)
    v = torch.randn(B, L, Hkv, D, generator=g, device="cuda").to(dtype)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dead = torch.arange(L, device="cuda")[None, :] >= lens[:, None]
    k[dead] = NAN
    v[dead] = NAN
    return q, k, v, lens, torch.rand(B, Hkv, L, generator=g, device="cuda")


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 13, 15, 16])
@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16)])
def test_keys_of_minus_infinity_leave_their_masses(G, D, dtype):
    """A key of -inf has weight exactly 0 for every number of heads per kv head, odd ones among them."""
    B, L, Hkv = 2, 300, 2
    q, k, v, lens, mass = make(B, L, Hkv, G, D, dtype, [300, 140], seed=G)
    q = q.abs() + 0.1
    gone = torch.zeros(L, dtype=torch.bool, device="cuda")
    gone[50:60] = True
    gone[129] = True
    k[:, gone] = -INF
    before = mass.clone()
    out, lse = cache_attention(q, k, v, lens, mass=mass)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all() and torch.isfinite(mass).all()
    assert torch.equal(mass[:, :, gone], before[:, :, gone])
    keep = (~gone).nonzero().flatten()
    fewer = torch.tensor([289, 129], dtype=torch.int32, device="cuda")
    ref.check_attention(out, lse, mass[..., keep], before[..., keep], q, k[:, keep], v[:, keep], fewer)


@pytest.mark.parametrize("D,dtype", [(64, FP16), (64, BF16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("G", [1, 4, 9])
def test_infinite_and_nan_values(G, D, dtype):
    """An infinite element of v makes its dimension infinite, with its sign, and no other; opposite
    infinities and NaN make it NaN: the products' own rules. The masses do not see v."""
    lens = [1, 40, 700, 333]
    q, k, v, lens, mass = make(4, 700, 2, G, D, dtype, lens, seed=D + G)
    _, clean_lse = cache_attention(q, k, v, lens, mass=(clean_mass := mass.clone()))
    v[0, 0, 0, 3] = INF
    v[1, 7, 1, 0], v[1, 39, 1, 0] = INF, INF
    v[1, 9, 0, D - 1] = -INF
    v[2, 650, 0, 5], v[2, 3, 0, 6], v[2, 699, 0, 6] = -INF, INF, -INF
    v[2, 333, 1, 17] = NAN
    out, lse = cache_attention(q, k, v, lens, mass=mass)
    assert torch.equal(lse, clean_lse) and torch.equal(mass, clean_mass)
    want = ref.attention(q, k, v, lens)[0].float()
    assert torch.equal(out.isnan(), want.isnan()), "NaN"
    assert torch.equal(out.isposinf(), want.isposinf()) and torch.equal(out.isneginf(), want.isneginf())
    finite = torch.where(v.isfinite(), v, 0.0)
    expect, _ = cache_attention(q, k, finite, lens)
    # Elsewhere the dimension does not know of it: fp32 sums in another order at most.
    ok = want.isfinite()
    err = (out.float() - expect.float()).abs()[ok]
    assert (err <= torch.finfo(dtype).eps * expect.float().abs()[ok] + 2.0 ** -15).all()
    assert _native.device_error() == 0


@pytest.mark.parametrize("D,dtype", [(64, FP16), (64, BF16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("G", [1, 3, 12])
@pytest.mark.parametrize("bits", [20, 26, 30])
def test_small_weights_beside_a_dominant_one(bits, G, D, dtype):
    """A first token that takes nearly all the weight and has values of 0, as attention sinks do: the
    output is the sum over the others, whose weights lie 2^-bits below."""
    L = 250
    g = torch.Generator(device="cuda").manual_seed(bits)
    q = torch.ones(1, G, D, device="cuda", dtype=dtype)
    k = (0.01 * torch.randn(1, L, 1, D, generator=g, device="cuda")).to(dtype)
    k[0, 0] = bits * math.log(2.0) / D ** 0.5
    v = (2000.0 * (1.0 + torch.rand(1, L, 1, D, generator=g, device="cuda"))).to(dtype)
    v[0, 0] = 0
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    out, lse = cache_attention(q, k, v, lens)
    want, rlse, _, absv, mag = ref.attention(q, k, v, lens)
    # Half a step of the output (fp16: or of its subnormals), and the weights' relative errors as in
    # cache_reference.check_attention. In fp16 the second part of a weight, 2^15 at most for the greatest, is a
    # multiple of 2^-24: the two parts are off by half of that, 2^-25 / 2^15 = 2^-40 of the greatest weight per
    # token, which is at most 1.
    half = torch.finfo(dtype).eps / 2
    tol = half * want.abs() + (2 * (D / 8 + 4) * 2.0 ** -24 * mag + 2.0 ** -19 + 2.0 ** -15)[..., None] * absv
    tol += 2.0 ** -25 + 2.0 ** -40 * v.double().abs().sum(1) if dtype == FP16 else torch.finfo(dtype).tiny
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3g} of the tolerance"


def test_sizes_past_a_c_int_are_refused():
    """2^32 + 4 tokens to keep are not 4, and a table of 2^32 + 1024 tokens is not one of 1024."""
    _, k, v, lens, mass = make(1, 64, 1, 1, 64, BF16, [64])
    outs = (torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lens), torch.zeros_like(mass))
    for budget in (2 ** 32 + 4, 2 ** 31 + 4, 2 ** 30 + 1):
        with pytest.raises(ValueError):
            cache_evict(k, v, lens, mass, *outs, budget)
    q, pool = torch.zeros(1, 1, 64, device="cuda").to(BF16), torch.zeros(2, 1024, 1, 64, device="cuda").to(BF16)
    table = torch.zeros(1, 2 ** 22 + 1, dtype=torch.int32, device="cuda")
    for out, lse in ((None, None), (torch.empty_like(q), torch.empty(1, 1, device="cuda"))):
        with pytest.raises(ValueError):
            cache_attention(q, pool, pool, lens, out, lse, block_table=table)
