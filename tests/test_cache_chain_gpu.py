"""Calls that follow one another on a stream without a pause, each on what the one before has just written (GPU)."""
import pytest
import torch

from fused_kernels_cutedsl_lib_b200 import cache_attention, cache_evict
from fused_kernels_cutedsl_lib_b200.layer import kv_append_paged

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("B,cap,budget", [(1, 256, 128), (6, 512, 200), (40, 128, 60), (3, 4096, 2000)])
def test_append_attend_evict_without_a_pause(B, cap, budget):
    """A decode loop in which the lengths, q, the cache, the masses, the partial results and the kept positions
    are each written by the kernel before: bit for bit the loop that waits after every call."""
    Hkv, G, D, page = 2, 4, 128, 16
    Hq, pages = Hkv * G, cap // page
    g = torch.Generator(device="cuda").manual_seed(B)
    qkvs = torch.randn(40, B, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(BF16)
    order = torch.randperm(2 * B * pages, generator=torch.Generator().manual_seed(B)).view(2, B, pages).int().cuda()
    first = torch.randint(0, cap - 40, (B,), generator=g, device="cuda").int()
    start = torch.randn(2 * B * pages, page, Hkv, D, generator=g, device="cuda").to(BF16)

    def loop(pause):
        k, v, tables = start.clone(), start.flip(0).contiguous(), order.clone()
        lens = [first.clone(), torch.zeros_like(first)]
        masses = [torch.zeros(B, Hkv, cap, device="cuda") for _ in range(2)]
        results, cur = [], 0
        torch.cuda.synchronize()
        for i, qkv in enumerate(qkvs):
            kv_append_paged(qkv, k, v, tables[cur], lens[cur], Hq, Hkv)
            pause()
            out, lse = cache_attention(qkv[:, :Hq * D].unflatten(1, (Hq, D)), k, v, lens[cur], block_table=tables[cur],
                                       mass=masses[cur])
            pause()
            results += [out, lse]
            if i % 8 == 5:
                results.append(cache_evict(k, v, lens[cur], masses[cur], k, v, lens[1 - cur], masses[1 - cur], budget,
                                           sinks=2, recent=8, block_table=tables[cur], out_block_table=tables[1 - cur]))
                pause()
                cur = 1 - cur
        torch.cuda.synchronize()
        return results + [k, v, *lens, *masses]

    want = loop(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(loop(lambda: None), want))
