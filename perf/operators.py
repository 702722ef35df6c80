"""Cases and plain forms of the memory-bound decode operators.

Three operators of a decode step whose HBM traffic is cut at both ends, the
weights and the KV cache:

* ``w4_linear``: y = x W^T (+ residual) for a few tokens, W held as 4-bit
  integers with a scale (and zero point) per group of input features;
* ``cache_attention``: softmax attention of one new token per sequence over a
  contiguous or paged KV cache (pages of any size), which also adds each cached
  token's attention weight to a running sum, its *mass*;
* ``cache_evict``: the tokens of least mass leave the cache; the kept ones, in
  order, are written to a smaller cache with their masses.

With ``own`` false, :func:`run` computes them from elementary torch operations
in fp32; with ``own`` true it calls this package. :func:`exact` restates the
definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    def w4(name, m, n, k, group, dtype="bf16", zeros=True, residual=False):
        return dict(name=name, op="w4", m=m, n=n, k=k, group=group, dtype=dtype, zeros=zeros, residual=residual)

    def attn(name, batch, lo, hi, page, hkv=8, g=4, d=128, dtype="bf16", mass=True, empty=0):
        return dict(name=name, op="attention", batch=batch, min_len=lo, max_len=hi, page=page, heads_kv=hkv, group=g,
                    dim=d, dtype=dtype, mass=mass, empty=empty)

    def evict(name, batch, lo, hi, budget, page, out_page, hkv=8, d=128, dtype="bf16", sinks=4, recent=64):
        return dict(name=name, op="evict", batch=batch, min_len=lo, max_len=hi, budget=budget, page=page,
                    out_page=out_page, heads_kv=hkv, dim=d, dtype=dtype, sinks=sinks, recent=recent)

    return [
        # One sequence answering: the attention output projection (+ residual) of a 4096-wide layer.
        w4("w4_o_proj_m1", 1, 4096, 4096, 128, residual=True),
        # The same step's fused QKV projection.
        w4("w4_qkv_m1", 1, 6144, 4096, 128),
        # Sixteen sequences through the gate/up projection, the widest weight of the layer.
        w4("w4_gate_up_m16", 16, 28672, 4096, 128),
        # A ragged vocabulary slice with small groups and no zero points, fp16.
        w4("w4_odd_m7_fp16", 7, 5003, 4000, 32, dtype="fp16", zeros=False),
        # A batch of 64 through the down projection: the largest token count a decode step sends here.
        w4("w4_down_m64", 64, 4096, 14336, 64, residual=True),
        # One short chat in a cache of 16-token pages: latency is all that counts.
        attn("attn_b1_l1000_page16", 1, 1000, 1000, 16, mass=False),
        # Four sequences in a padded contiguous cache, masses kept for a later eviction.
        attn("attn_b4_l4096", 4, 4096, 4096, 0),
        # Small heads, one query head in three sharing, odd pages, rows that hold nothing yet.
        attn("attn_odd_b17_d64_fp16", 17, 1, 2311, 24, hkv=5, g=3, d=64, dtype="fp16", empty=2),
        # A full serving batch with lengths from 512 to 32768: bandwidth is all that counts.
        attn("attn_ragged_b64_l32768", 64, 512, 32768, 64),
        # Small odd caches, some already below the budget; paged to contiguous.
        evict("evict_odd_b6_d64_fp16", 6, 300, 2311, 777, 24, 0, hkv=5, d=64, dtype="fp16", sinks=3, recent=31),
        # One long prompt cut to a short cache: eight heads' selections over 32768 tokens, latency.
        evict("evict_b1_l32768_to_2048", 1, 32768, 32768, 2048, 16, 16),
        # A whole batch cut to 4096 tokens each: the copy of the kept rows is what costs.
        evict("evict_ragged_b32_to_4096", 32, 512, 32768, 4096, 64, 64, recent=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["w4", "attention", "evict"])
    if op == "w4":
        group = rng.choice([32, 64, 128])
        while True:
            c = dict(op=op, m=_log_int(rng, 1, 64), n=_log_int(rng, 200, 28672),
                     k=group * _log_int(rng, max(1, 256 // group), 14336 // group), group=group,
                     dtype=rng.choice(["bf16", "fp16"]), zeros=rng.random() < 0.6, residual=rng.random() < 0.4)
            if c["m"] * c["n"] * c["k"] <= 64 * 4096 * 14336 and c["n"] * c["k"] <= 28672 * 4096:
                return c
    page = rng.choice([0, 16, 64, rng.randint(1, 130)])
    if op == "attention":
        while True:
            hi = _log_int(rng, 16, 32768)
            batch = _log_int(rng, 1, 64)
            c = dict(op=op, batch=batch, min_len=rng.randint(0, hi), max_len=hi, page=page,
                     heads_kv=rng.choice([1, 2, 3, 4, 8]), group=rng.choice([1, 2, 4, 5, 7, 8, 12, 16]),
                     dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "fp16"]), mass=rng.random() < 0.7,
                     empty=rng.choice([0, 0, min(batch - 1, 1)]))
            c["heads_kv"] = min(c["heads_kv"], 32 // c["group"]) or 1
            w = work(c)
            if w["bytes"] <= 4.4e9 and w["flops"] <= 17.8e9:
                return c
    while True:
        hi = _log_int(rng, 64, 32768)
        budget = _log_int(rng, 8, max(8, hi - 1))
        recent = rng.randint(0, budget // 2)
        c = dict(op=op, batch=_log_int(rng, 1, 32), min_len=rng.randint(0, hi), max_len=hi, budget=budget, page=page,
                 out_page=rng.choice([0, page, rng.randint(1, 100)]), heads_kv=rng.choice([1, 2, 4, 5, 8]),
                 dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "fp16"]),
                 sinks=rng.randint(0, min(16, budget - recent)), recent=recent)
        if work(c)["bytes"] <= 1.0e9:
            return c


def _lengths(case):
    """Cache lengths of the batch: spread evenly over [min_len, max_len] (the seed only orders them),
    `empty` rows holding nothing."""
    b, e = case["batch"], case.get("empty", 0)
    lo, hi = case["min_len"], case["max_len"]
    lens = [lo + (hi - lo) * (i + 1) // b for i in range(b)]
    return [0] * e + lens[e:]


def work(case):
    if case["op"] == "w4":
        m, n, k, gr = case["m"], case["n"], case["k"], k_groups(case)
        nbytes = n * k / 2 + n * gr * 2 + (n * gr if case["zeros"] else 0) + 2 * m * (k + n * (2 if case["residual"] else 1))
        return {"bytes": nbytes, "flops": 2.0 * m * n * k}
    lens, hkv, d = _lengths(case), case["heads_kv"], case["dim"]
    tokens = sum(lens)
    pages = 4 * sum(-(-x // case["page"]) for x in lens) if case["page"] else 0
    if case["op"] == "attention":
        hq = hkv * case["group"]
        nbytes = tokens * hkv * d * 4 + case["batch"] * (hq * (4 * d + 4) + 4) + pages
        if case["mass"]:
            nbytes += 8 * tokens * hkv
        return {"bytes": nbytes, "flops": 4.0 * tokens * hq * d}
    kept = sum(min(x, case["budget"]) for x in lens)
    cap = case["budget"]
    nbytes = (4 * tokens * hkv + 8 * kept * hkv * d + case["batch"] * hkv * cap * 8 + 8 * case["batch"] + pages)
    if case["out_page"]:
        nbytes += 4 * sum(-(-min(x, cap) // case["out_page"]) for x in lens)
    return {"bytes": nbytes, "flops": 0.0}


def k_groups(case):
    return case["k"] // case["group"]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "w4":
        st = _prepare_w4(case, gen)
        if own:
            # The weight's layout for the kernel, made once when a model is loaded.
            from fused_kernels_cutedsl_lib_b200 import pack_w4

            st["weight"] = pack_w4(st["q"], st["scales"], st["zeros"])
    elif case["op"] == "attention":
        st = _prepare_attention(case, gen, seed)
        if own:
            from fused_kernels_cutedsl_lib_b200 import alloc_cache_attention_workspace

            st["workspace"] = alloc_cache_attention_workspace(
                case["batch"], st["capacity"], case["heads_kv"] * case["group"], case["heads_kv"], case["dim"],
                mass=case["mass"], device="cuda")
    else:
        st = _prepare_evict(case, gen, seed)
    st["case"] = case
    return st


def _prepare_w4(case, gen):
    dt = DTYPES[case["dtype"]]
    m, n, k, gr = case["m"], case["n"], case["k"], k_groups(case)
    # Quantised normal weights: bell-shaped codes, zero points around the middle, scales that give the
    # dequantised weight a standard deviation near 0.02; activations with a few large channels.
    q = (torch.randn(n, k, generator=gen, device="cuda", dtype=torch.bfloat16) * 2.6 + 7.5).round_().clamp_(0, 15)
    scales = (0.004 + 0.008 * torch.rand(n, gr, generator=gen, device="cuda")).to(dt)
    zeros = torch.randint(5, 11, (n, gr), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    x = torch.randn(m, k, generator=gen, device="cuda")
    x[:, ::97] *= 8.0
    residual = torch.randn(m, n, generator=gen, device="cuda").to(dt) if case["residual"] else None
    return dict(q=q.to(torch.uint8), scales=scales, zeros=zeros, x=x.to(dt), residual=residual,
                out=torch.empty(m, n, device="cuda", dtype=dt))


def _pages(lens, page, cap_pages, seed):
    """A block table [B, cap_pages] over shuffled physical pages, and the pool's size in pages."""
    need = [-(-x // page) for x in lens]
    order = np.random.RandomState(seed % (1 << 31)).permutation(sum(need) + 1)
    table, at = np.zeros((len(lens), cap_pages), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), sum(need) + 1


def _cache(case, gen, seed, lens):
    """(k, v, block table or None, capacity in tokens per row): random rows in the valid places and
    whatever is left in the rest."""
    dt, hkv, d, page = DTYPES[case["dtype"]], case["heads_kv"], case["dim"], case["page"]
    longest = max(1, case["max_len"])
    if page:
        table, pool = _pages(lens, page, -(-longest // page), seed)
        shape, cap = (pool, page, hkv, d), -(-longest // page) * page
    else:
        table, shape, cap = None, (case["batch"], longest, hkv, d), longest
    k = torch.empty(shape, device="cuda", dtype=dt).normal_(generator=gen)
    v = torch.empty(shape, device="cuda", dtype=dt).normal_(generator=gen)
    return k, v, table, cap


def _prepare_attention(case, gen, seed):
    lens = np.random.RandomState(seed % (1 << 31)).permutation(_lengths(case)).astype(np.int32)
    k, v, table, cap = _cache(case, gen, seed, lens.tolist())
    dt, hkv, hq, d = DTYPES[case["dtype"]], case["heads_kv"], case["heads_kv"] * case["group"], case["dim"]
    b = case["batch"]
    # Queries a little wider than the keys, so that some tokens carry most of the weight.
    q = (1.5 * torch.randn(b, hq, d, generator=gen, device="cuda")).to(dt)
    mass = torch.rand(b, hkv, cap, generator=gen, device="cuda") if case["mass"] else None
    return dict(q=q, k=k, v=v, table=table, capacity=cap, lens=torch.from_numpy(lens).cuda(), mass=mass,
                mass_out=torch.zeros_like(mass) if case["mass"] else None,
                out=torch.empty(b, hq, d, device="cuda", dtype=dt), lse=torch.empty(b, hq, device="cuda"))


def _prepare_evict(case, gen, seed):
    lens = np.random.RandomState(seed % (1 << 31)).permutation(_lengths(case)).astype(np.int32)
    k, v, table, cap = _cache(case, gen, seed, lens.tolist())
    b, hkv, d, budget, page = case["batch"], case["heads_kv"], case["dim"], case["budget"], case["out_page"]
    # Attention masses: a long tail of heavy tokens, and tokens that no step has looked at yet.
    mass = torch.randn(b, hkv, cap, generator=gen, device="cuda").mul_(2.0).exp_()
    mass *= torch.rand(b, hkv, cap, generator=gen, device="cuda") > 0.1
    if page:
        out_table, pool = _pages([budget] * b, page, -(-budget // page), seed + 1)
        shape, out_cap = (pool, page, hkv, d), -(-budget // page) * page
    else:
        out_table, shape, out_cap = None, (b, budget, hkv, d), budget
    k_out = torch.zeros(shape, device="cuda", dtype=k.dtype)
    return dict(k=k, v=v, table=table, capacity=cap, lens=torch.from_numpy(lens).cuda(), mass=mass, k_out=k_out,
                v_out=torch.zeros_like(k_out), out_table=out_table, out_capacity=out_cap,
                mass_out=torch.zeros(b, hkv, out_cap, device="cuda"),
                lens_out=torch.zeros(b, dtype=torch.int32, device="cuda"),
                kept=torch.zeros(b, hkv, budget, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if c["op"] == "w4":
        return _own_w4(st) if own else _plain_w4(st)
    if c["op"] == "attention":
        return _own_attention(st) if own else _plain_attention(st)
    return _own_evict(st) if own else _plain_evict(st)


def _own_w4(st):
    from fused_kernels_cutedsl_lib_b200 import w4_linear

    return w4_linear(st["x"], st["weight"], st["out"], residual=st["residual"])


def _own_attention(st):
    from fused_kernels_cutedsl_lib_b200 import cache_attention

    cache_attention(st["q"], st["k"], st["v"], st["lens"], st["out"], st["lse"], block_table=st["table"],
                    mass=st["mass"], mass_out=st["mass_out"], workspace=st["workspace"])
    return _attention_outputs(st["out"], st["lse"], st["mass_out"])


def _own_evict(st):
    from fused_kernels_cutedsl_lib_b200 import cache_evict

    c = st["case"]
    cache_evict(st["k"], st["v"], st["lens"], st["mass"], st["k_out"], st["v_out"], st["lens_out"], st["mass_out"],
                c["budget"], sinks=c["sinks"], recent=c["recent"], block_table=st["table"],
                out_block_table=st["out_table"], kept=st["kept"])
    return _evict_outputs(st["k_out"], st["v_out"], st["mass_out"], st["lens_out"], st["kept"])


def _attention_outputs(out, lse, mass):
    r = {"out": out, "lse": lse}
    if mass is not None:
        r["mass"] = mass
    return r


def _evict_outputs(k, v, mass, lens, kept):
    return {"k": k, "v": v, "mass": mass, "lens": lens, "kept": kept}


def _plain_w4(st):
    c = st["case"]
    n, k, gr = c["n"], c["k"], k_groups(c)
    q = st["q"].view(n, gr, c["group"]).float()
    z = 8.0 if st["zeros"] is None else st["zeros"].float()[:, :, None]
    w = ((q - z) * st["scales"].float()[:, :, None]).view(n, k)
    y = st["x"].float() @ w.t()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(st["out"].dtype)


def _rows_of(cache, table, cap):
    """The cache as [B, capacity, heads, dim] in token order."""
    if table is None:
        return cache
    return cache[table.long()].flatten(1, 2)[:, :cap]


def _plain_attention(st):
    c = st["case"]
    b, hkv, g, d, cap = c["batch"], c["heads_kv"], c["group"], c["dim"], st["capacity"]
    valid = torch.arange(cap, device="cuda")[None, :] < st["lens"][:, None]  # [B, cap]
    q = st["q"].float().view(b, hkv, g, d)
    k = _rows_of(st["k"], st["table"], cap).float().permute(0, 2, 3, 1)
    s = (q @ k) / math.sqrt(d)
    del k
    s = s.masked_fill(~valid[:, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - top.clamp_min(-1e30)).exp()
    total = e.sum(-1, keepdim=True)
    lse = (top + total.log()).view(b, hkv * g)
    p = e / total.clamp_min(1e-30)
    v = _rows_of(st["v"], st["table"], cap).float().permute(0, 2, 1, 3)
    v = v.masked_fill(~valid[:, None, :, None], 0.0)
    out = (p @ v).view(b, hkv * g, d).to(st["out"].dtype)
    mass = None
    if c["mass"]:
        mass = torch.where(valid[:, None, :], st["mass"] + p.sum(2), st["mass_out"])
    return _attention_outputs(out, lse, mass)


def _plain_evict(st):
    c = st["case"]
    b, hkv, cap, budget = c["batch"], c["heads_kv"], st["capacity"], c["budget"]
    lens = st["lens"].long()
    at = torch.arange(cap, device="cuda")
    n = lens[:, None, None]
    protected = (at < c["sinks"]) | (at >= n - c["recent"])
    # Protected tokens before all others, then by mass; places behind the end come last. The sort is stable.
    key = st["mass"].masked_fill(protected, math.inf).masked_fill(at >= n, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    if cap < budget:
        order = torch.cat([order, torch.full((b, hkv, budget - cap), cap, device="cuda")], -1)
    new = lens.clamp_max(budget)
    slot = torch.arange(budget, device="cuda")
    live = (slot < new[:, None, None]).expand(b, hkv, budget)
    kept = torch.where(live, order[:, :, :budget], cap).sort(-1).values
    src = kept.clamp_max(cap - 1)
    head = torch.arange(hkv, device="cuda")[None, :, None]
    mass = torch.zeros_like(st["mass_out"])
    mass[:, :, :budget] = st["mass"].gather(-1, src).masked_fill(~live, 0.0)
    from_row = _physical(src, st["table"], c["page"], cap)
    to_row = _physical(slot.expand(b, hkv, budget), st["out_table"], c["out_page"], budget)
    outs = []
    for name in ("k", "v"):
        old = st[name + "_out"].flatten(0, 1)
        rows = torch.where(live[..., None], st[name].flatten(0, 1)[from_row, head], old[to_row, head])
        moved = old.clone()
        moved[to_row, head] = rows
        outs.append(moved.view(st[name + "_out"].shape))
    kept = torch.where(live, kept, -1).to(torch.int32)
    return _evict_outputs(outs[0], outs[1], mass, new.to(torch.int32), kept)


def _physical(pos, table, page, cap):
    """Row of the flattened cache that holds token `pos` [B, heads, n] of each sequence."""
    b = torch.arange(pos.shape[0], device="cuda")[:, None, None]
    if table is None:
        return b * cap + pos
    return table.long()[b, pos // page] * page + pos % page


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "w4":
        w = st["q"].double()
        w -= 8.0 if st["zeros"] is None else st["zeros"].double().repeat_interleave(case["group"], dim=1)
        w *= st["scales"].double().repeat_interleave(case["group"], dim=1)
        y = torch.einsum("mk,nk->mn", st["x"].double(), w)
        return y if st["residual"] is None else y + st["residual"].double()
    if case["op"] == "attention":
        return _exact_attention(case, st)
    return _exact_evict(case, st)


def _exact_attention(case, st):
    hkv, g, d = case["heads_kv"], case["group"], case["dim"]
    b = case["batch"]
    out = torch.zeros(b, hkv * g, d, device="cuda", dtype=torch.float64)
    lse = torch.full((b, hkv * g), -math.inf, device="cuda", dtype=torch.float64)
    mass = st["mass_out"].double() if case["mass"] else None
    for i, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        if st["table"] is None:
            k, v = st["k"][i, :n], st["v"][i, :n]
        else:
            at = torch.arange(n, device="cuda")
            page, row = st["table"][i].long()[at // case["page"]], at % case["page"]
            k, v = st["k"][page, row], st["v"][page, row]
        for h in range(hkv):
            s = torch.einsum("gd,td->gt", st["q"][i, h * g:(h + 1) * g].double(), k[:, h].double()) * d ** -0.5
            z = torch.logsumexp(s, 1)
            w = torch.exp(s - z[:, None])
            lse[i, h * g:(h + 1) * g] = z
            out[i, h * g:(h + 1) * g] = torch.einsum("gt,td->gd", w, v[:, h].double())
            if mass is not None:
                mass[i, h, :n] = st["mass"][i, h, :n].double() + w.sum(0)
    return _attention_outputs(out, lse, mass)


def _exact_evict(case, st):
    """Which tokens stay, by an ordinary sort of (mass, place) per head; the copied rows themselves are
    not computed values."""
    mass, lens = st["mass"].cpu().numpy(), st["lens"].tolist()
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    kept = np.full((case["batch"], case["heads_kv"], budget), -1, np.int32)
    out = np.zeros(tuple(st["mass_out"].shape), np.float64)
    for i, n in enumerate(lens):
        for h in range(case["heads_kv"]):
            if n <= budget:
                keep = np.arange(n)
            else:
                middle = np.arange(sinks, n - recent)
                best = middle[np.lexsort((middle, -mass[i, h, sinks:n - recent]))[:budget - sinks - recent]]
                keep = np.concatenate([np.arange(sinks), np.sort(best), np.arange(n - recent, n)])
            kept[i, h, :len(keep)] = keep
            out[i, h, :len(keep)] = mass[i, h, keep]
    new = np.minimum(np.asarray(lens), budget).astype(np.int32)
    return _evict_outputs(None, None, out, new, kept)
