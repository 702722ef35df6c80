"""Plain 64-bit forms of cache attention with mass and of eviction, and seeded caches (test helpers)."""
import math

import torch


def page_in(k, v, page, spare=2, seed=0, extra_pages=1):
    """The contiguous caches [B, L, H, D] scattered over shuffled pages: (k_pool, v_pool, table).
    Every row gets ``extra_pages`` table entries past its capacity that name a page of NaN."""
    B, L, H, D = k.shape
    n = -(-L // page)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(B * n + spare, generator=g)
    pools = []
    for c in (k, v):
        pool = torch.full((B * n + spare, page, H, D), float("nan"), dtype=c.dtype, device=c.device)
        pad = torch.full((B, n * page, H, D), float("nan"), dtype=c.dtype, device=c.device)
        pad[:, :L] = c
        pool[order[:B * n].to(c.device)] = pad.view(B * n, page, H, D)
        pools.append(pool)
    table = torch.full((B, n + extra_pages), int(order[-1]), dtype=torch.int32)
    table[:, :n] = order[:B * n].view(B, n).int()
    return pools[0], pools[1], table.to(k.device)


def attention(q, k, v, lens, scale=None):
    """(out, lse, weights [B, Hkv, L] summed over the group) in float64, one row at a time, and the
    bounds that tolerances need: sum w |v| [B, Hq, D] and max |q||k| scale per row and head [B, Hq]."""
    B, Hq, D = q.shape
    L, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    dev = q.device
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=dev)
    absv = torch.zeros_like(out)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=dev)
    mag = torch.zeros(B, Hq, dtype=torch.float64, device=dev)
    w_sum = torch.zeros(B, Hkv, L, dtype=torch.float64, device=dev)
    for b, n in enumerate(lens.clamp(0, L).tolist()):
        for h in range(Hkv if n else 0):
            rows = slice(h * G, (h + 1) * G)
            qq, kk, vv = q[b, rows].double(), k[b, :n, h].double(), v[b, :n, h].double()
            s = qq @ kk.t() * scale
            w = torch.softmax(s, -1)
            lse[b, rows] = torch.logsumexp(s, -1)
            out[b, rows] = w @ vv
            absv[b, rows] = w @ vv.abs()
            mag[b, rows] = (qq.abs() @ kk.abs().t()).amax(-1) * abs(scale)
            w_sum[b, h, :n] = w.sum(0)
    return out, lse, w_sum, absv, mag


def check_attention(out, lse, mass_out, mass, q, k, v, lens, scale=None):
    """Tolerances, with u = 2^-24 the unit of fp32: a score is off by at most
    ds = (D/8 + 4) u max sum |q||k| scale (two units of the magnitude per 16-wide mma step, and
    the scaling); a weight then by a factor of 1 +- (2 ds + 2^-19) (exponentials, the running
    maximum's rescaling, sums of up to 2^16 terms split over lanes, warps and splits); P enters the
    second product as two 16-bit numbers, 2^-16 together for bf16; the output is rounded once."""
    ref, rlse, rw, absv, mag = attention(q, k, v, lens, scale)
    D = q.shape[-1]
    ds = (D / 8 + 4) * 2.0 ** -24 * mag
    rel = 2 * ds + 2.0 ** -19
    half = torch.finfo(out.dtype).eps / 2
    tol = half * ref.abs() + (rel + 2.0 ** -15)[..., None] * absv + torch.finfo(out.dtype).tiny
    err = (out.double().view_as(ref) - ref).abs()
    assert (err <= tol).all(), f"out: worst {(err / tol).nan_to_num(9e9).max().item():.3g} of the tolerance"
    empty = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    e = (lse.double() - rlse).abs()[~empty]
    assert (e <= (rel + 2.0 ** -22 * (1 + rlse.abs()))[~empty]).all(), f"lse: {e.max().item():.3g}"
    if mass_out is None:
        return
    L, Hkv = k.shape[1], k.shape[2]
    live = torch.arange(L, device=q.device)[None, None, :] < lens.clamp(0, L)[:, None, None]
    relh = rel.view(q.shape[0], Hkv, -1).amax(-1)[..., None]
    want = torch.where(live, mass[..., :L].double() + rw, mass[..., :L].double())
    e = (mass_out[..., :L].double() - want).abs()
    assert (e <= relh * rw + 2.0 ** -23 * want.abs()).all(), f"mass: {e.max().item():.3g}"


def evict(k, v, lens, mass, budget, sinks, recent):
    """(kept [B, H, budget] with -1 behind, new lengths) by a stable sort per head."""
    B, L, H, _ = k.shape
    kept = torch.full((B, H, budget), -1, dtype=torch.int32)
    new = lens.clamp(0, L).clamp_max(budget)
    for b, n in enumerate(lens.clamp(0, L).tolist()):
        for h in range(H):
            if n <= budget:
                idx = torch.arange(n)
            else:
                mid = mass[b, h, sinks:n - recent].cpu()
                best = torch.sort(mid, descending=True, stable=True).indices[:budget - sinks - recent] + sinks
                idx = torch.cat([torch.arange(sinks), best.sort().values, torch.arange(n - recent, n)])
            kept[b, h, :len(idx)] = idx.int()
    return kept.to(k.device), new


def rows(cache, table, b, n):
    """The first n tokens of row b of a contiguous (table None) or paged cache, [n, H, D]."""
    if table is None:
        return cache[b, :n]
    page = cache.shape[1]
    at = torch.arange(n, device=cache.device)
    return cache[table[b].long()[at // page], at % page]
