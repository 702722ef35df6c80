"""Cache attention with mass, and eviction by mass, against plain 64-bit forms (GPU)."""
import pytest
import torch

import cache_reference as ref
from fused_kernels_cutedsl_lib_b200 import (
    _native,
    alloc_cache_attention_workspace,
    cache_attention,
    cache_evict,
    decode_attention,
    pack_w4,
    w4_linear,
)
from fused_kernels_cutedsl_lib_b200.layer import kv_append, kv_append_paged

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
NAN = float("nan")


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
    mass = torch.rand(B, Hkv, L + 3, generator=g, device="cuda")
    return q, k, v, lens, mass


def run(q, k, v, lens, mass=None, **kw):
    out = torch.full_like(q, NAN)
    lse = torch.full(q.shape[:2], NAN, device="cuda")
    mass_out = None
    if mass is not None:
        mass_out = torch.full_like(mass, -7.0)
    cache_attention(q, k, v, lens, out, lse, mass=mass, mass_out=mass_out, **kw)
    torch.cuda.synchronize()
    return out, lse, mass_out


CASES = [
    # B, L, Hkv, G, lens
    (1, 1, 1, 1, [1]),
    (1, 64, 2, 4, [64]),
    (3, 130, 2, 3, [0, 1, 130]),
    (4, 300, 1, 8, [63, 64, 65, 299]),
    (2, 1000, 3, 5, [1000, 17]),
    (5, 200, 2, 16, [200, 0, 199, 128, 129]),
    (2, 2500, 8, 12, [2500, 1201]),
    (40, 333, 4, 2, [(37 * i) % 334 for i in range(40)]),
    (2, 9000, 1, 9, [9000, 4097]),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}L{c[1]}H{c[2]}G{c[3]}")
def test_attention_matches_definition(case, D, dtype):
    B, L, Hkv, G, lens = case
    q, k, v, lens, mass = make(B, L, Hkv, G, D, dtype, lens, seed=B + L)
    got = run(q, k, v, lens, mass)
    ref.check_attention(got[0], got[1], None, None, q, k, v, lens)
    live = torch.arange(L + 3, device="cuda")[None, None] < lens[:, None, None]
    assert (got[2].masked_select(~live.expand_as(mass)) == -7.0).all()  # behind the lengths: as it was
    ref.check_attention(got[0], got[1], torch.where(live, got[2], mass), mass, q, k, v, lens)
    plain = run(q, k, v, lens)
    assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])
    for page in (1, 7, 16, 24, 64, 100):
        kp, vp, table = ref.page_in(k, v, page, seed=page)
        paged = run(q, kp, vp, lens, torch.nn.functional.pad(mass, (0, 400)), block_table=table)
        # Another capacity gives other splits: the same values within the tolerance.
        padded = torch.where(live, paged[2][..., :L + 3], mass)
        ref.check_attention(paged[0], paged[1], padded, mass, q, k, v, lens)
    assert _native.device_error() == 0


def test_attention_agrees_with_decode_attention():
    q, k, v, lens, _ = make(3, 700, 4, 4, 128, BF16, [700, 1, 345], seed=2)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    out, lse = cache_attention(q, k, v, lens)
    other, olse = decode_attention(q, k, v, lens)
    # decode_attention rounds P to bf16 (2^-8 of weights that sum to 1, |v| < 6) and both round the output.
    assert (out.float() - other.view_as(out).float()).abs().max().item() <= 2 * 6 * 2.0 ** -8
    assert (lse - olse).abs().max().item() <= 1e-4


def test_attention_mass_in_place_and_repeated_bits():
    q, k, v, lens, mass = make(6, 500, 2, 4, 128, BF16, [500, 0, 3, 257, 64, 100], seed=4)
    first = run(q, k, v, lens, mass)
    m = mass.clone()
    out, lse = cache_attention(q, k, v, lens, mass=m)
    live = torch.arange(503, device="cuda")[None, None] < lens[:, None, None]
    assert torch.equal(m, torch.where(live, first[2], mass))
    for _ in range(10):
        again = run(q, k, v, lens, mass)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_attention_strided_q_lengths_out_of_range_and_scale():
    B, L, Hkv, G, D = 4, 150, 2, 4, 128
    q, k, v, lens, mass = make(B, L, Hkv, G, D, BF16, [150, 150, 0, 70], seed=5)
    wide = torch.randn(B, (Hkv * G + 2 * Hkv) * D, device="cuda").to(BF16)
    view = wide[:, :Hkv * G * D].view(B, Hkv * G, D)
    view.copy_(q)
    told = torch.tensor([150, 9999, -4, 70], dtype=torch.int32, device="cuda")  # clamped to [0, 150]
    for scale in (None, 0.5, -0.03, 0.0):
        out, lse = cache_attention(view, k, v, told, softmax_scale=scale)
        ref.check_attention(out, lse, None, None, q, k, v, lens, scale=scale)
        out4, _ = cache_attention(view.unsqueeze(1), k, v, told, softmax_scale=scale)
        assert torch.equal(out, out4)


def test_attention_extreme_scores():
    """A dominant token, scores of the type's extremes, and -inf scores."""
    q, k, v, lens, mass = make(3, 200, 1, 2, 64, BF16, [200, 200, 200], seed=6)
    k[0, 123] = 40.0 * q[0, 0] / q[0, 0].norm()
    k[1] = 0
    got = run(q, k, v, lens, mass)
    ref.check_attention(got[0], got[1], torch.where(got[2] == -7.0, mass, got[2]), mass, q, k, v, lens)
    # A K row of -inf where q is positive: weight exactly 0 and no NaN anywhere.
    q[2] = q[2].abs() + 0.1
    k[2, 50:60] = float("-inf")
    out, lse, m = run(q, k, v, lens, mass)
    assert torch.isfinite(out[2]).all() and torch.isfinite(lse[2]).all()
    assert torch.equal(m[2, 0, 50:60], mass[2, 0, 50:60])
    keep = torch.tensor([i for i in range(200) if not 50 <= i < 60], device="cuda")
    ref.check_attention(out[2:], lse[2:], None, None, q[2:], k[2:, keep], v[2:, keep], lens[2:] - 10)
    # All scores -inf: the kernels' convention of an empty row. A NaN key makes its heads NaN.
    k[2] = float("-inf")
    out, lse, m = run(q, k, v, lens, mass)
    assert (out[2] == 0).all() and torch.isinf(lse[2]).all() and torch.equal(m[2, 0, :200], mass[2, 0, :200])
    k[1, 77] = NAN
    out, lse, _ = run(q, k, v, lens)
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all() and torch.isfinite(out[0]).all()


def test_attention_pages_outside_the_pool_read_as_zeros():
    q, k, v, lens, mass = make(2, 64, 2, 4, 128, BF16, [64, 50], seed=7)
    kp, vp, table = ref.page_in(k, v, 16)
    bad = table.clone()
    bad[0, 1], bad[1, 2] = -1, kp.shape[0]
    k2, v2 = k.clone(), v.clone()
    k2[0, 16:32], v2[0, 16:32] = 0, 0
    k2[1, 32:48], v2[1, 32:48] = 0, 0
    got = run(q, kp, vp, lens, torch.nn.functional.pad(mass, (0, 40)), block_table=bad)
    ref.check_attention(got[0], got[1], None, None, q, k2, v2, lens)


def test_attention_streams_graphs_and_workspaces():
    q, k, v, lens, mass = make(4, 600, 2, 4, 128, FP16, [600, 1, 320, 599], seed=8)
    want = run(q, k, v, lens, mass)
    ws = alloc_cache_attention_workspace(4, 600, 8, 2, 128, mass=True)
    ws.fill_(255)
    got = run(q, k, v, lens, mass, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    side = torch.cuda.Stream()
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    side.wait_stream(torch.cuda.current_stream())
    cache_attention(q, k, v, lens, out, lse, stream=side)
    side.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    # Two graphs without a workspace argument, replayed at the same time on two streams.
    graphs = []
    for _ in range(2):
        o, l, m = torch.empty_like(out), torch.empty_like(lse), mass.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                cache_attention(q, k, v, lens, o, l, mass=m)
        graphs.append((g, o, l, m))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (g, *_), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    m = mass.clone()
    for _ in range(15):
        cache_attention(q, k, v, lens, mass=m)
    for _, o, l, mm in graphs:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1]) and torch.equal(mm, m)


def test_attention_offsets_past_32_bits():
    """Pages at the far end of a pool of more than 2^32 elements."""
    Hkv, D, page, pages = 8, 128, 64, 70000
    kp = torch.empty(pages, page, Hkv, D, dtype=BF16, device="cuda")
    vp = torch.empty(pages, page, Hkv, D, dtype=BF16, device="cuda")
    assert kp.numel() > 1 << 32
    q, k, v, lens, mass = make(1, 128, Hkv, 4, D, BF16, [100], seed=9)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    kp[table[0].long()] = k[0].view(2, page, Hkv, D)
    vp[table[0].long()] = v[0].view(2, page, Hkv, D)
    got = run(q, kp, vp, lens, mass, block_table=table)
    ref.check_attention(got[0], got[1], None, None, q, k, v, lens)
    # Evicted into other far pages of the same pools.
    out_table = torch.tensor([[pages - 2]], dtype=torch.int32, device="cuda")
    new, m2 = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1, Hkv, 64), NAN, device="cuda")
    kept = cache_evict(kp, vp, lens, mass, kp, vp, new, m2, 40, sinks=2, recent=5, block_table=table,
                       out_block_table=out_table)
    want, n = ref.evict(k, v, lens, mass, 40, 2, 5)
    assert torch.equal(kept, want) and int(new) == 40
    idx = kept[0].long().t()
    heads = torch.arange(Hkv, device="cuda")[None]
    assert torch.equal(kp[pages - 2, :40], k[0][idx, heads]) and torch.equal(vp[pages - 2, :40], v[0][idx, heads])


def check_evict(k, v, lens, mass, budget, sinks, recent, table=None, out_page=0, extra_out=5, src=None):
    """One call, everything it writes compared; k, v contiguous reference, src the caches really passed."""
    B, L, H, D = k.shape
    ck, cv = (k, v) if src is None else src
    need = min(budget, L if table is None else table.shape[1] * ck.shape[1])
    if out_page:
        n = -(-need // out_page)
        out_table = torch.randperm(B * n + 1)[:B * n].view(B, n).int().cuda()
        shape = (B * n + 1, out_page, H, D)
    else:
        out_table, shape = None, (B, need + extra_out, H, D)
    ko, vo = torch.full(shape, 3.0, dtype=k.dtype, device="cuda"), torch.full(shape, 5.0, dtype=k.dtype, device="cuda")
    new = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    m_out = torch.full((B, H, need + extra_out), NAN, device="cuda")
    kept = torch.full((B, H, budget), -9, dtype=torch.int32, device="cuda")
    got = cache_evict(ck, cv, lens, mass, ko, vo, new, m_out, budget, sinks=sinks, recent=recent, block_table=table,
                      out_block_table=out_table, kept=kept)
    torch.cuda.synchronize()
    assert got is kept
    want, n_new = ref.evict(k, v, lens, mass, budget, sinks, recent)
    assert torch.equal(kept, want)
    assert torch.equal(new, n_new.int())
    heads = torch.arange(H, device="cuda")[None]
    touched = torch.zeros(shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(n_new.tolist()):
        idx = kept[b, :, :n].long().t()  # [n, H]
        assert torch.equal(ref.rows(ko, out_table, b, n).view(torch.int16), k[b][idx, heads].view(torch.int16))
        assert torch.equal(ref.rows(vo, out_table, b, n).view(torch.int16), v[b][idx, heads].view(torch.int16))
        gathered = mass[b].gather(1, kept[b, :, :n].long())
        assert torch.equal(m_out[b, :, :n].view(torch.int32), gathered.view(torch.int32))
        assert (m_out[b, :, n:] == 0).all()
        at = torch.arange(n, device="cuda")
        if out_table is None:
            touched[b, :n] = True
        else:
            touched[out_table[b].long()[at // out_page], at % out_page] = True
    assert (ko[~touched] == 3.0).all() and (vo[~touched] == 5.0).all()
    return kept


EVICT = [
    # B, L, H, lens, budget, sinks, recent
    (1, 1, 1, [1], 1, 0, 0),
    (1, 2, 1, [2], 1, 0, 0),
    (3, 40, 2, [0, 40, 7], 8, 2, 3),
    (2, 100, 3, [100, 99], 100, 4, 10),
    (2, 100, 3, [100, 99], 99, 4, 10),
    (4, 1000, 1, [1000, 600, 33, 500], 32, 0, 32),
    (4, 1000, 2, [1000, 600, 33, 500], 32, 32, 0),
    (2, 1000, 2, [1000, 36], 35, 3, 31),
    (2, 5000, 2, [5000, 4097], 1025, 0, 0),
    (1, 40000, 2, [39999], 4096, 4, 256),
    (33, 700, 5, [(97 * i) % 701 for i in range(33)], 250, 5, 17),
    (1, 70, 1, [70], 200, 5, 17),
]


@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16)])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"B{c[0]}L{c[1]}H{c[2]}budget{c[4]}s{c[5]}r{c[6]}")
def test_evict_matches_definition(case, D, dtype):
    B, L, H, lens, budget, sinks, recent = case
    _, k, v, lens, mass = make(B, L, H, 1, D, dtype, lens, seed=L + budget)
    mass *= torch.rand_like(mass) > 0.3  # many equal masses of 0
    check_evict(k, v, lens, mass, budget, sinks, recent)
    for page, out_page in ((1, 3), (16, 0), (24, 16), (64, 64)):
        kp, vp, table = ref.page_in(k, v, page, seed=page)
        cap = table.shape[1] * page
        padded = torch.nn.functional.pad(mass[..., :L], (0, max(0, cap - L)), value=1e9)
        check_evict(k, v, lens, padded, budget, sinks, recent, table=table, out_page=out_page, src=(kp, vp))


def test_evict_masses_equal_signed_infinite_and_nan():
    _, k, v, lens, mass = make(2, 3000, 2, 1, 64, BF16, [3000, 2999], seed=11)
    for value in (0.0, 1.5, float("inf")):
        mass.fill_(value)
        kept = check_evict(k, v, lens, mass, 100, 3, 7)
        assert kept[0, 0, 3:93].tolist() == list(range(3, 93))  # ties go to the earliest
    mass = torch.randint(-3, 3, mass.shape, device="cuda").float()
    check_evict(k, v, lens, mass, 777, 3, 7)
    mass[:, :, ::2] *= -0.0  # both zeros are one value
    check_evict(k, v, lens, mass, 777, 3, 7)
    mass[:, :, 5::11] = float("inf")
    mass[:, :, 6::11] = float("-inf")
    mass[:, :, 7::301] = NAN  # greatest, as torch.sort has it
    check_evict(k, v, lens, mass, 777, 3, 7)
    mass = torch.randn(mass.shape, device="cuda").exp() * 1e-38  # subnormals among them
    check_evict(k, v, lens, mass, 777, 0, 0)


def test_evict_graph_stream_and_same_pool():
    _, k, v, lens, mass = make(2, 320, 2, 1, 128, BF16, [320, 310], seed=12)
    kp, vp, table = ref.page_in(k, v, 32, spare=8, extra_pages=0)
    used = set(table.flatten().tolist())
    free = [i for i in range(kp.shape[0]) if i not in used]
    out_table = torch.tensor(free[:8], dtype=torch.int32, device="cuda").view(2, 4)
    new, m2 = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 128, device="cuda")
    kept = torch.zeros(2, 2, 100, dtype=torch.int32, device="cuda")
    args = (kp, vp, lens, mass, kp, vp, new, m2, 100)
    kw = dict(sinks=4, recent=20, block_table=table, out_block_table=out_table, kept=kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache_evict(*args, stream=side, **kw)
    side.synchronize()
    want, _ = ref.evict(k, v, lens, mass, 100, 4, 20)
    heads = torch.arange(2, device="cuda")[None]

    def check(want):
        assert torch.equal(kept, want)
        for b in range(2):
            idx = want[b].long().t()
            assert torch.equal(ref.rows(kp, out_table, b, 100), k[b][idx, heads])

    check(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_evict(*args, **kw)
    mass.copy_(torch.rand_like(mass))
    graph.replay()
    torch.cuda.synchronize()
    check(ref.evict(k, v, lens, mass, 100, 4, 20)[0])


def test_evict_pages_outside_the_pool():
    """A bad input page reads as zero rows, a bad output page is not written."""
    _, k, v, lens, mass = make(1, 64, 2, 1, 64, BF16, [64], seed=13)
    kp, vp, table = ref.page_in(k, v, 16, extra_pages=0)
    table[0, 1] = kp.shape[0] + 5
    ko, vo = torch.full((3, 16, 2, 64), 9.0, dtype=BF16, device="cuda"), torch.full((3, 16, 2, 64), 9.0, dtype=BF16, device="cuda")
    out_table = torch.tensor([[2, -1, 0]], dtype=torch.int32, device="cuda")
    new, m2 = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, 48, device="cuda")
    kept = cache_evict(kp, vp, lens, mass, ko, vo, new, m2, 40, recent=40 - 1, block_table=table,
                       out_block_table=out_table)
    torch.cuda.synchronize()
    k2 = k[0].clone()
    k2[16:32] = 0
    idx, heads = kept[0].long().t(), torch.arange(2, device="cuda")[None]
    assert torch.equal(ko[2], k2[idx[:16], heads]) and torch.equal(ko[0, :8], k2[idx[32:], heads])
    assert (ko[1] == 9.0).all() and (ko[0, 8:] == 9.0).all()


def test_decode_with_a_bounded_cache():
    """The operators as a decode loop uses them: 4-bit projections around attention over a cache that
    is evicted whenever it is full, against the same loop in plain 64-bit steps on the same caches."""
    torch.manual_seed(3)
    B, Hkv, G, D, page, cap, budget = 3, 2, 4, 128, 16, 96, 48
    Hq, hidden = Hkv * G, 256
    qkv_dim = (Hq + 2 * Hkv) * D

    def weight(n, k):
        q = torch.randint(0, 16, (n, k), dtype=torch.uint8, device="cuda")
        s = (0.002 + 0.008 * torch.rand(n, k // 64, device="cuda")).to(BF16)
        z = torch.randint(5, 11, (n, k // 64), dtype=torch.uint8, device="cuda")
        w = pack_w4(q, s, z)
        return w, w.dequantize().double()

    w_qkv, d_qkv = weight(qkv_dim, hidden)
    w_o, d_o = weight(hidden, Hq * D)
    pages = cap // page
    pool_k = torch.zeros(2 * B * pages, page, Hkv, D, dtype=BF16, device="cuda")
    pool_v = torch.zeros_like(pool_k)
    tables = torch.randperm(2 * B * pages).view(2, B, pages).int().cuda()
    lens = torch.tensor([0, 90, 41], dtype=torch.int32, device="cuda")
    # Rows that already hold a prompt.
    for b, n in enumerate(lens.tolist()):
        at = torch.arange(n, device="cuda")
        pool_k[tables[0, b].long()[at // page], at % page] = torch.randn(n, Hkv, D, device="cuda").to(BF16)
        pool_v[tables[0, b].long()[at // page], at % page] = torch.randn(n, Hkv, D, device="cuda").to(BF16)
    mass = torch.rand(B, Hkv, cap, device="cuda")
    live = torch.arange(cap, device="cuda")[None, None] < lens[:, None, None]
    mass *= live
    spare_mass, spare_lens = torch.zeros_like(mass), torch.zeros_like(lens)
    cur, evictions = 0, 0
    for step in range(120):
        if step % 12 == 6:  # a server evicts between steps, before the longest row is full
            table, new = tables[cur], tables[1 - cur]
            old_k = torch.stack([ref.rows(pool_k, table, b, cap) for b in range(B)])
            want, n_new = ref.evict(old_k, old_k, lens, mass, budget, 2, 8)
            kept = cache_evict(pool_k, pool_v, lens, mass, pool_k, pool_v, spare_lens, spare_mass, budget, sinks=2,
                               recent=8, block_table=table, out_block_table=new)
            assert torch.equal(kept, want) and torch.equal(spare_lens, n_new.int())
            lens, spare_lens, mass, spare_mass, cur = spare_lens, lens, spare_mass, mass, 1 - cur
            evictions += 1
        table = tables[cur]
        x = torch.randn(B, hidden, device="cuda").to(BF16)
        qkv = w4_linear(x, w_qkv)
        kv_append_paged(qkv, pool_k, pool_v, table, lens, Hq, Hkv)
        before = mass.clone()
        out, lse = cache_attention(qkv[:, :Hq * D].unflatten(1, (Hq, D)), pool_k, pool_v, lens, block_table=table,
                                   mass=mass)
        y = w4_linear(out.view(B, -1), w_o, residual=x)
        if step % 20 == 7:
            want_qkv = x.double() @ d_qkv.t()
            assert ((qkv.double() - want_qkv).norm() / want_qkv.norm()).item() <= 2.0 ** -8
            k = torch.stack([ref.rows(pool_k, table, b, cap) for b in range(B)])
            v = torch.stack([ref.rows(pool_v, table, b, cap) for b in range(B)])
            q = qkv[:, :Hq * D].reshape(B, Hq, D)
            ref.check_attention(out, lse, mass, before, q, k, v, lens)
            want_y = out.view(B, -1).double() @ d_o.t() + x.double()
            assert ((y.double() - want_y).norm() / want_y.norm()).item() <= 2.0 ** -8
    assert evictions == 10 and lens.tolist() == [54, 54, 54]


def test_contiguous_cache_appends_after_eviction():
    """The masses behind the new lengths are zero, so that appended tokens start from nothing."""
    B, Hkv, G, D, cap = 2, 2, 4, 128, 80
    _, k, v, lens, mass = make(B, cap, Hkv, 1, D, BF16, [80, 30], seed=15)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    new, m2 = torch.zeros_like(lens), torch.full((B, Hkv, cap), NAN, device="cuda")
    cache_evict(k, v, lens, mass, ko, vo, new, m2, 40, sinks=1, recent=4)
    qkv = torch.randn(B, (Hkv * G + 2 * Hkv) * D, device="cuda").to(BF16)
    kv_append(qkv, ko, vo, new, Hkv * G, Hkv)
    assert new.tolist() == [41, 31]
    before = m2.clone()
    q = qkv[:, :Hkv * G * D].unflatten(1, (Hkv * G, D))
    out, lse = cache_attention(q, ko, vo, new, mass=m2)
    ref.check_attention(out, lse, m2, before, q.reshape(B, -1, D), ko, vo, new)
    assert (before[0, :, 40] == 0).all() and (m2[0, :, 40] > 0).all() and (m2[0, :, 41:] == 0).all()


def test_refusals():
    q, k, v, lens, mass = make(2, 64, 2, 4, 128, BF16, [64, 10], seed=16)
    ok = lambda **kw: cache_attention(kw.pop("q", q), kw.pop("k", k), kw.pop("v", v), kw.pop("lens", lens), **kw)  # noqa: E731
    ok()
    with pytest.raises(TypeError):
        ok(q=q.float())
    with pytest.raises(TypeError):
        ok(k=k.half())
    with pytest.raises(TypeError):
        ok(lens=lens.long())
    for bad in (dict(q=q[:, :3]), dict(q=q[:1]), dict(k=k[:, :32]), dict(k=k[..., :64], v=v[..., :64]),
                dict(lens=lens[:1]), dict(k=k.transpose(1, 2), v=v.transpose(1, 2)), dict(mass=mass[:, :1]),
                dict(mass=torch.zeros(2, 2, 63, device="cuda")), dict(mass_out=mass), dict(softmax_scale=NAN),
                dict(block_table=torch.zeros(1, 2, dtype=torch.int32, device="cuda")),
                dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                dict(out=torch.empty(2, 8, 64, dtype=BF16, device="cuda"))):
        with pytest.raises(ValueError):
            ok(**bad)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    new, m2 = torch.zeros_like(lens), torch.zeros_like(mass)

    def ev(k_out=ko, v_out=vo, seqlens_out=new, mass_out=m2, budget=32, **kw):
        return cache_evict(k, v, lens, mass, k_out, v_out, seqlens_out, mass_out, budget, **kw)

    ev()
    for bad in (dict(budget=0), dict(sinks=-1), dict(recent=33), dict(sinks=20, recent=20), dict(k_out=k, v_out=v),
                dict(v_out=ko), dict(seqlens_out=lens), dict(mass_out=mass), dict(k_out=ko[:, :16].contiguous(),
                v_out=vo[:, :16].contiguous()), dict(mass_out=torch.zeros(2, 2, 31, device="cuda")),
                dict(kept=torch.zeros(2, 2, 31, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            ev(**bad)


# Long rows of few heads: more stretches of a row than a warp has lanes, several times over.
@pytest.mark.parametrize("B,L,Hkv,G,lens", [(1, 40000, 1, 4, [39999]), (2, 33000, 1, 16, [33000, 1]),
                                            (1, 70000, 2, 1, [65537])])
@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16)])
def test_attention_long_rows(B, L, Hkv, G, lens, D, dtype):
    q, k, v, lens, mass = make(B, L, Hkv, G, D, dtype, lens, seed=L)
    got = run(q, k, v, lens, mass)
    live = torch.arange(L + 3, device="cuda")[None, None] < lens[:, None, None]
    ref.check_attention(got[0], got[1], torch.where(live, got[2], mass), mass, q, k, v, lens)
    assert (got[2].masked_select(~live.expand_as(mass)) == -7.0).all()


# More masses per lane than the other sizes have, and more than a lane's registers hold.
@pytest.mark.parametrize("B,L,H,D,lens,budget", [(20, 20000, 8, 8, [20000 - 997 * i for i in range(20)], 3000),
                                                 (1, 300000, 2, 16, [300000], 5000), (1, 270001, 1, 8, [262145], 262144)])
def test_evict_long_rows(B, L, H, D, lens, budget):
    _, k, v, lens, mass = make(B, L, H, 1, D, BF16, lens, seed=L)
    mass *= torch.rand_like(mass) > 0.3
    check_evict(k, v, lens, mass, budget, 4, 60)


def test_mass_may_not_overlap_itself():
    q, k, v, lens, _ = make(2, 64, 2, 4, 128, BF16, [64, 10], seed=21)
    flat = torch.zeros(2 * 2 * 64 + 2 * 64, device="cuda")
    mass, shifted = flat[:256].view(2, 2, 64), flat[128:384].view(2, 2, 64)
    with pytest.raises(ValueError):
        cache_attention(q, k, v, lens, mass=mass, mass_out=shifted)
    cache_attention(q, k, v, lens, mass=mass, mass_out=flat[:256].view(2, 2, 64))  # the same memory: in place
    assert (flat[256:] == 0).all()


def test_evictions_on_two_streams_at_once():
    sets = []
    for seed in (31, 32):
        _, k, v, lens, mass = make(6, 3000, 2, 1, 64, BF16, [3000, 0, 77, 1500, 513, 2999], seed=seed)
        want, new = ref.evict(k, v, lens, mass, 512, 4, 32)
        out = [torch.empty(6, 512, 2, 64, dtype=BF16, device="cuda") for _ in range(2)]
        sets.append((k, v, lens, mass, out, torch.empty_like(lens), torch.empty(6, 2, 512, device="cuda"), want,
                     torch.empty_like(want), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for k, v, lens, mass, out, new, m, want, kept, st in sets:
            cache_evict(k, v, lens, mass, *out, new, m, 512, sinks=4, recent=32, kept=kept, stream=st)
    torch.cuda.synchronize()
    for k, v, lens, mass, out, new, m, want, kept, st in sets:
        assert torch.equal(kept, want)
