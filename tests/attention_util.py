"""Plain 64-bit forms of the operators between a decode step's projections, and the error bounds their tests use."""
import math

import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}      # half of the smallest step near zero


def paged_cache(lens, kv, dim, page, dtype, dev, seed=0, spare=3, width=None, heads_first=False):
    """Caches of NaN with only the tokens of `lens` filled in, a table of shuffled pages (unused entries: far outside the cache)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    width = max(1, max(need, default=0)) if width is None else width
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)
    shape = (pages, kv, page, dim) if heads_first else (pages, page, kv, dim)
    k, v = (torch.full(shape, math.nan, dtype=DT[dtype]) for _ in range(2))
    kt, vt = (t.transpose(1, 2) if heads_first else t for t in (k, v))
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            name = int(order[at])
            at += 1
            if i < width:
                table[b, i] = name
            live = min(page, n - i * page)
            kt[name, :live] = torch.randn((live, kv, dim), generator=g).to(DT[dtype])
            vt[name, :live] = torch.randn((live, kv, dim), generator=g).to(DT[dtype])
    k, v = k.to(dev), v.to(dev)
    return (k.transpose(1, 2), v.transpose(1, 2), table.to(dev)) if heads_first else (k, v, table.to(dev))


def attend(q, k, v, table, lens, scale, window, cap):
    """(out, lse, bound on |out - computed|, bound on |lse - computed|) in 64 bits, on the CPU.

    Worst case of fp32 arithmetic with u = 2^-24: a score is a sum of D products (D + 4 roundings of partial sums no larger than
    sum |q k|, the tensor cores may cut instead of round: twice that), so a weight is off by 2 x that, by the exponential (2^-21) and
    by the roundings of the running sums over n keys, each no larger than n u (again twice) of sum p |v|; a weight kept as
    two 16-bit parts loses at most 2^-16 of itself.  The rounding of the output comes on top in the caller."""
    u2 = 2.0 ** -23
    q, k, v, table = (t.detach().cpu() for t in (q, k, v, table))
    (b, h, d), (pages, page, kv, _) = q.shape, k.shape
    out, lse = torch.zeros(b, h, d, dtype=torch.float64), torch.full((b, h), -math.inf, dtype=torch.float64)
    eo, el = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lens):
        n0 = max(n, 0)
        js = [j for j in range(max(0, n0 - window) if window else 0, min(n0, table.shape[1] * page)) if 0 <= int(table[i, j // page]) < pages]
        if not js:
            continue
        names = torch.tensor([int(table[i, j // page]) for j in js])
        place = torch.tensor([j % page for j in js])
        kk = k[names, place].double().repeat_interleave(h // kv, 1)          # [n, h, d]
        vv = v[names, place].double().repeat_interleave(h // kv, 1)
        s = torch.einsum("hd,nhd->hn", q[i].double(), kk) * scale
        es = (d + 4) * u2 * scale * torch.einsum("hd,nhd->hn", q[i].double().abs(), kk.abs()).amax(1)
        if cap:
            s = cap * torch.tanh(s / cap)
            es = es + cap * 2.0 ** -21
        norm = torch.logsumexp(s, 1)
        p = torch.exp(s - norm[:, None])
        out[i], lse[i] = torch.einsum("hn,nhd->hd", p, vv), norm
        es = es + u2 * s.abs().amax(1)
        rel = torch.expm1(2 * es) + 2.0 ** -16 + 2.0 ** -20 + 2 * len(js) * u2
        eo[i] = rel[:, None] * torch.einsum("hn,nhd->hd", p, vv.abs())
        el[i] = es + 2.0 ** -20 + len(js) * u2 + 4 * u2 * norm.abs()
    return out, lse, eo, el


def check_attention(got, want, bound, dtype):
    got = got.detach().double().cpu()
    assert bool(torch.isfinite(got).all())
    limit = bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * want.abs() + TINY[dtype]
    off = (got - want).abs()
    assert bool((off <= limit).all()), float((off / limit.clamp_min(1e-300)).max())


def rotate(x, positions, inv_freq, w, eps, interleaved, factor):
    """x [tokens, heads, D] -> (result, bound on the fp32 error) in 64 bits."""
    x = x.detach().cpu().double()
    size = x.abs()
    if w is not None:
        inv = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
        x, size = x * inv * w.detach().cpu().double(), size * inv * w.detach().cpu().double().abs()
    half = inv_freq.numel()
    ang = positions.detach().cpu().double()[:, None, None] * inv_freq.detach().cpu().double()
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, e = x.clone(), size.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    e[..., a] = (size[..., a] + size[..., b]) * abs(factor)
    e[..., b] = (size[..., a] + size[..., b]) * abs(factor)
    # mean of D squares and its root: (D + 6) u; weight, factor, product and sum: 8 u; cosine and sine of an angle in [-pi, pi]
    # rounded to fp32: 2^-23 in the angle and 2 ulp of the functions
    return y, e * ((x.shape[-1] + 14) * 2.0 ** -24 + 2.0 ** -21)


def route(logits, top_k, scoring, bias, groups, top_groups, renormalize, scale):
    """(weights, ids) in 64 bits with Python's own sorting: best first, ties to the lowest index."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), torch.tensor(-math.inf, dtype=torch.float64), x).clamp_max(3.4028234663852886e38)
    weights, ids = [], []
    for row in x:
        if scoring == "sigmoid":
            p = torch.sigmoid(row)
        else:
            ex = torch.exp(row - row.max().clamp_min(-3.4e38))
            p = ex / ex.sum().clamp_min(1e-300)
        c = (row if bias is None else p + bias.detach().cpu().double()).tolist()
        size = len(c) // groups
        allowed = range(len(c))
        if groups > 1:
            runs = [sorted(c[g * size:(g + 1) * size], reverse=True) for g in range(groups)]
            value = [r[0] if bias is None else sum(r[:2]) for r in runs]
            kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
            allowed = [e for g in sorted(kept) for e in range(g * size, (g + 1) * size)]
        pick = sorted(allowed, key=lambda e: (-c[e], e))[:top_k]
        w = p[pick]
        if renormalize:
            w = w / w.sum().clamp_min(1e-300)
        weights.append(w * scale)
        ids.append(pick)
    return torch.stack(weights), torch.tensor(ids, dtype=torch.int32)


def pages(table, seen, new, free, taken, page, num_tokens):
    """What plan_pages returns, in Python: (table, total, starts, positions, slots, taken)."""
    table, width = [row[:] for row in table], len(table[0]) if table else 0
    starts, positions, slots = [0], [], []
    for r, (s, n) in enumerate(zip(seen, new)):
        s, n = max(s, 0), max(n, 0)
        held = -(-s // page)
        for at in range(held, min(-(-(s + n) // page), width)):
            table[r][at] = free[taken] if taken < len(free) else -1
            taken += 1
        for pos in range(s, s + n):
            name = table[r][pos // page] if pos // page < width else -1
            positions.append(pos)
            slots.append(name * page + pos % page if name >= 0 else -1)
        starts.append(starts[-1] + n)
    pad = num_tokens - len(positions)
    return table, [max(s, 0) + max(n, 0) for s, n in zip(seen, new)], starts, positions + [0] * pad, slots + [-1] * pad, taken
