"""The operators between the projections of a decode step, as a serving program calls them: query/key norms with the position
rotation (and the cache write), attention of one new token over a paged cache, page tables and slots from request lengths, and
the routing of tokens to experts.

`own` chooses between the package's entry points (`kaillm_b200.attention`, `kaillm_b200.linear.route_experts`) and a plain form
made of elementary torch operations.  `work` counts every input read once and every output written once.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_KV = 64 * 8192 * 8 * 128 * 2      # cached values (keys and values) of the largest listed attention
MOST_QK = 64 * 8192 * 40 * 128         # score products of the largest listed attention
MOST_ROWS = 8192 * 56 * 128            # values of the largest listed rotation
TINY = 1.1754943508222875e-38          # smallest normal fp32


def listed():
    return [
        # one user, a short chat turn: a few hundred cached tokens, latency
        {"name": "attend_1seq_200", "kind": "attend", "seqs": 1, "low": 200, "high": 200, "heads": 40, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "cap": 0.0, "lse": False, "dtype": "bf16"},
        # one user, a long document: the work of one sequence has to fill the GPU
        {"name": "attend_1seq_128k", "kind": "attend", "seqs": 1, "low": 131071, "high": 131071, "heads": 40, "kv": 8, "dim": 128,
         "page": 16, "window": 0, "cap": 0.0, "lse": True, "dtype": "f16"},
        # a decode batch of ordinary lengths, and one of many users with lengths from nothing to 16k
        {"name": "attend_16seq_2k", "kind": "attend", "seqs": 16, "low": 900, "high": 3100, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "cap": 0.0, "lse": False, "dtype": "bf16"},
        {"name": "attend_64seq_16k", "kind": "attend", "seqs": 64, "low": 0, "high": 16384, "heads": 40, "kv": 8, "dim": 128, "page": 64,
         "window": 0, "cap": 0.0, "lse": False, "dtype": "bf16"},
        # wide heads, all of them sharing two key heads, a sliding window and capped scores, single precision
        {"name": "attend_window_f32", "kind": "attend", "seqs": 33, "low": 100, "high": 7001, "heads": 16, "kv": 2, "dim": 256, "page": 32,
         "window": 1024, "cap": 50.0, "lse": False, "dtype": "f32"},
        # a token of a decode step into the cache; a batch of them without norms and with interleaved pairs, partly rotated; a prefill chunk
        {"name": "rotate_1tok", "kind": "rotate", "tokens": 1, "heads": 40, "kv": 8, "dim": 128, "rotated": 128, "interleaved": False,
         "norm": True, "store": True, "page": 16, "far": 131072, "dtype": "bf16"},
        {"name": "rotate_partial_61tok", "kind": "rotate", "tokens": 61, "heads": 32, "kv": 2, "dim": 128, "rotated": 64, "interleaved": True,
         "norm": False, "store": False, "page": 16, "far": 1000000, "dtype": "f32"},
        {"name": "rotate_8192tok", "kind": "rotate", "tokens": 8192, "heads": 40, "kv": 8, "dim": 128, "rotated": 128, "interleaved": False,
         "norm": True, "store": True, "page": 16, "far": 40000, "dtype": "bf16"},
        # page tables and slots of a decode step, and of a batch of prompts
        {"name": "pages_decode_64", "kind": "pages", "requests": 64, "seen": 20000, "new": 1, "page": 16},
        {"name": "pages_prompts_500", "kind": "pages", "requests": 500, "seen": 0, "new": 1050, "page": 32},
        # routing of a decode batch, and of a prefill chunk with a balancing bias and groups
        {"name": "route_8tok", "kind": "route", "tokens": 8, "experts": 128, "top_k": 8, "scoring": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "renormalize": True, "scale": 1.0, "dtype": "bf16"},
        {"name": "route_16384tok", "kind": "route", "tokens": 16384, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "rotate", "rotate", "pages", "route", "route"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    heads, kv = rng.choice(((40, 8), (16, 8), (20, 20), (64, 8), (28, 4), (8, 1), (71, 1), (6, 2)))
    dim = rng.choice((64, 80, 128, 128, 256))
    if kind == "attend":
        seqs = _log(rng, 1, 256)
        # cached tokens of the whole batch: as many bytes and score products as the largest listed case at most
        most = min(MOST_KV // (kv * dim * 2) // (2 if dtype == "f32" else 1), MOST_QK // (heads * dim), 262144)
        high = _log(rng, 1, min(131072, max(1, most // seqs)))
        low = rng.choice((0, 1, high // 2, high))
        return {"kind": kind, "seqs": seqs, "low": min(low, high), "high": high, "heads": heads, "kv": kv, "dim": dim,
                "page": rng.choice((16, 16, 32, 64, 48, 128)), "window": rng.choice((0, 0, 0, 128, 1000, 4096)),
                "cap": rng.choice((0.0, 0.0, 0.0, 30.0)), "lse": rng.random() < 0.25, "dtype": dtype}
    if kind == "rotate":
        tokens = _log(rng, 1, max(1, min(8192, MOST_ROWS // ((heads + 2 * kv) * dim) // (2 if dtype == "f32" else 1))))
        return {"kind": kind, "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "rotated": rng.choice((dim, dim, dim, dim // 2)),
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7, "store": rng.random() < 0.6, "page": rng.choice((16, 32, 48)),
                "far": _log(rng, 100, 1000000), "dtype": dtype}
    if kind == "pages":
        requests = _log(rng, 1, 2048)
        new = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, 262144 // requests))
        return {"kind": kind, "requests": requests, "seen": rng.choice((0, _log(rng, 1, 32768))), "new": new, "page": rng.choice((16, 32, 48, 128))}
    experts = rng.choice((8, 32, 60, 64, 128, 160, 256, 384, 512))
    groups = rng.choice((1, 1, 4, 8)) if experts in (32, 64, 128, 160, 256) else 1
    top_groups = max(1, groups // 2)
    return {"kind": kind, "tokens": _log(rng, 1, 16384 * 256 // max(256, experts)), "experts": experts,
            "top_k": rng.choice([k for k in (1, 2, 4, 6, 8, 10) if k <= experts // groups * top_groups]),
            "scoring": rng.choice(("softmax", "sigmoid")), "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
            "renormalize": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5)), "dtype": dtype}


def _spread(n, lo, hi):
    """n whole numbers spread evenly from lo to hi."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _generator(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _normal(shape, dtype, g, dev):
    """Made in the type itself: a large cache needs no temporaries."""
    out = torch.empty(shape, dtype=DTYPES[dtype], device=dev)
    return out.normal_(generator=g)


def _shuffled(values, g, dev):
    t = torch.tensor(values, dtype=torch.int32, device=dev)
    return t[torch.randperm(len(values), generator=g, device=dev)]


def _inv_freq(rotated, dev):
    return (1e6 ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)).to(torch.float32).to(dev)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = _generator(seed, dev)
    if case["kind"] == "attend":
        lens = _shuffled(_spread(case["seqs"], case["low"], case["high"]), g, dev)
        held = (lens.long() + case["page"] - 1) // case["page"]
        width = max(1, -(-case["high"] // case["page"]))
        total = sum(-(-n // case["page"]) for n in _spread(case["seqs"], case["low"], case["high"]))
        pages = total + 3
        # pages were handed out in the order in which the sequences grew: no sequence's pages lie together
        order = torch.randperm(pages, generator=g, device=dev)[:total].to(torch.int32)
        column = torch.arange(width, device=dev)
        mine = column < held[:, None]
        table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=dev)
        table[mine] = order
        shape = (pages, case["page"], case["kv"], case["dim"])
        q = _normal((case["seqs"], case["heads"], case["dim"]), case["dtype"], g, dev) * 1.5
        return {"kind": "attend", "q": q, "k": _normal(shape, case["dtype"], g, dev), "v": _normal(shape, case["dtype"], g, dev),
                "table": table, "lens": lens, "scale": case["dim"] ** -0.5, "window": case["window"], "cap": case["cap"], "lse": case["lse"]}
    if case["kind"] == "rotate":
        t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
        state = {"kind": "rotate", "heads": h, "kv": kv, "interleaved": case["interleaved"], "store": case["store"],
                 "qkv": _normal((t, (h + 2 * kv) * d), case["dtype"], g, dev) * 2.0,
                 "positions": torch.randint(0, case["far"], (t,), generator=g, device=dev, dtype=torch.int32),
                 "inv_freq": _inv_freq(case["rotated"], dev), "qw": None, "kw": None}
        if case["norm"]:
            state["qw"], state["kw"] = _normal((d,), case["dtype"], g, dev) * 0.2 + 1, _normal((d,), case["dtype"], g, dev) * 0.2 + 1
        if case["store"]:
            pages = -(-t // case["page"]) + 2
            shape = (pages, case["page"], kv, d)
            state["kc"], state["vc"] = _normal(shape, case["dtype"], g, dev), _normal(shape, case["dtype"], g, dev)
            state["slots"] = torch.randperm(pages * case["page"], generator=g, device=dev)[:t]
            if t > 8:
                state["slots"][t - 1] = -1     # a padded batch
        return state
    if case["kind"] == "pages":
        r, page = case["requests"], case["page"]
        seen = _shuffled(_spread(r, 0, case["seen"]), g, dev)
        new = torch.full((r,), 1, dtype=torch.int32, device=dev) if case["new"] == 1 else _shuffled(_spread(r, 0, case["new"]), g, dev)
        width = -(-(case["seen"] + case["new"]) // page) + 1
        held = (seen + page - 1) // page
        names = torch.randperm(r * width, generator=g, device=dev).to(torch.int32)
        table = torch.where(torch.arange(width, device=dev, dtype=torch.int32) < held[:, None], names.view(r, width), -1)
        return {"kind": "pages", "table": table.contiguous(), "seen": seen, "new": new, "page": page,
                "free": torch.randperm(r * width + 5, generator=g, device=dev).to(torch.int32) + r * width,
                "taken": torch.tensor([3], dtype=torch.int32, device=dev), "tokens": _tokens(case)}
    logits = _normal((case["tokens"], case["experts"]), case["dtype"], g, dev) * 1.5
    bias = torch.randn(case["experts"], generator=g, device=dev) * 0.1 if case["bias"] else None
    return {"kind": "route", "logits": logits, "bias": bias, "top_k": case["top_k"], "scoring": case["scoring"], "groups": case["groups"],
            "top_groups": case["top_groups"], "renormalize": case["renormalize"], "scale": case["scale"]}


def _tokens(case):
    """Entries of the slot list: the new tokens, padded to a multiple of eight as a captured step's batch is."""
    new = case["requests"] if case["new"] == 1 else sum(_spread(case["requests"], 0, case["new"]))
    return max(8, -(-new // 8) * 8)


def _attend(q, k_cache, v_cache, table, lens, scale, window, cap, lse):
    (b, h, d), (_, page, kv, _) = q.shape, k_cache.shape
    at = torch.arange(table.shape[1] * page, device=q.device)
    live = (at < lens[:, None]) & ((at >= lens[:, None] - window) if window else True)                  # [b, n]
    slot = (table.long().clamp_min(0) * page)[:, at // page] + at % page
    k = k_cache.view(-1, kv, d)[slot].float().permute(0, 2, 3, 1)                                         # [b, kv, d, n]
    s = torch.matmul(q.float().view(b, kv, h // kv, d), k) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    s = s.masked_fill(~live[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    v = v_cache.view(-1, kv, d)[slot].float().masked_fill(~live[:, :, None, None], 0).permute(0, 2, 1, 3)
    o = (torch.matmul(e, v) / total.clamp_min(TINY)).view(b, h, d).to(q.dtype)
    return (o, (top + torch.log(total)).view(b, h)) if lse else o


def _turn(x, cos, sin, interleaved):
    """x [t, heads, d] in 32 bits; cos, sin [t, r / 2]."""
    half = cos.shape[1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _rotate(qkv, positions, inv_freq, heads, kv, qw, kw, interleaved, k_cache=None, v_cache=None, slots=None):
    t, dt = qkv.shape[0], qkv.dtype
    x = qkv.view(t, heads + 2 * kv, -1)
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = x[:, :heads].float(), x[:, heads:heads + kv].float()
    if qw is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * qw.float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * kw.float()
    q, k = _turn(q, cos, sin, interleaved).to(dt), _turn(k, cos, sin, interleaved).to(dt)
    if slots is None:
        return q, k
    keep = slots >= 0
    k_cache.view(-1, kv, k.shape[-1])[slots[keep]] = k[keep]
    v_cache.view(-1, kv, k.shape[-1])[slots[keep]] = x[:, heads + kv:][keep]
    return q, k_cache, v_cache


def _pages(table, seen, new, free, taken, page, tokens):
    width = table.shape[1]
    held, total = (seen + page - 1) // page, seen + new
    need = ((total + page - 1) // page).clamp_max(width) - held
    first = taken + torch.cumsum(need, 0) - need
    column = torch.arange(width, device=table.device, dtype=torch.int32)
    fresh = (column >= held[:, None]) & (column < (held + need)[:, None])
    at = first[:, None] + column - held[:, None]
    table.copy_(torch.where(fresh, torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1), table))
    starts = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0)).to(torch.int32)
    t = torch.arange(tokens, device=table.device, dtype=torch.int32)
    r = torch.searchsorted(starts[1:], t, right=True)
    real = r < seen.numel()
    r = r.clamp_max(seen.numel() - 1)
    positions = torch.where(real, seen[r] + t - starts[r], 0).to(torch.int32)
    name = table[r, (positions // page).clamp_max(width - 1)].long()
    slots = torch.where(real & (positions < width * page) & (name >= 0), name * page + positions % page, -1)
    return table, total, starts, positions, slots, (taken + need.sum()).to(torch.int32)


def _route(logits, top_k, scoring, bias, groups, top_groups, renormalize, scale):
    t, e = logits.shape
    x = logits.float()
    p = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    # the choice: in the order of the logits without a bias, otherwise in 64 bits, where scores next to each other stay apart
    wide = logits.double()
    c = wide if bias is None else (torch.softmax(wide, -1) if scoring == "softmax" else torch.sigmoid(wide)) + bias.double()
    if groups > 1:
        g = c.view(t, groups, e // groups)
        best = g.amax(-1) if bias is None else torch.sort(g, dim=-1, descending=True)[0][..., :2].sum(-1)
        chosen = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :top_groups]
        keep = torch.zeros((t, groups), dtype=torch.bool, device=x.device).scatter_(1, chosen, True)
        c = g.masked_fill(~keep[:, :, None], -math.inf).view(t, e)
    ids = torch.sort(c, dim=-1, descending=True, stable=True)[1][:, :top_k]
    w = p.gather(1, ids)
    if renormalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(TINY)
    return w * scale, ids.to(torch.int32)


def run(state):
    s = state
    if own:
        from kaillm_b200 import attention, linear
        if s["kind"] == "attend":
            return attention.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], scale=s["scale"], window=s["window"],
                                             softcap=s["cap"], return_lse=s["lse"])
        if s["kind"] == "rotate":
            if s["store"]:
                q = attention.qk_norm_rope_store(s["qkv"], s["positions"], s["inv_freq"], s["heads"], s["kc"], s["vc"], s["slots"],
                                                 q_weight=s["qw"], k_weight=s["kw"], interleaved=s["interleaved"])
                return q, s["kc"], s["vc"]
            return attention.qk_norm_rope(s["qkv"], s["positions"], s["inv_freq"], s["heads"], s["kv"], q_weight=s["qw"], k_weight=s["kw"],
                                          interleaved=s["interleaved"])
        if s["kind"] == "pages":
            return s["table"], *attention.plan_pages(s["table"], s["seen"], s["new"], s["free"], s["taken"], s["page"], s["tokens"])
        return linear.route_experts(s["logits"], s["top_k"], scoring=s["scoring"], bias=s["bias"], groups=s["groups"],
                                    top_groups=s["top_groups"], renormalize=s["renormalize"], scale=s["scale"])
    if s["kind"] == "attend":
        return _attend(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], s["window"], s["cap"], s["lse"])
    if s["kind"] == "rotate":
        cache = (s["kc"], s["vc"], s["slots"]) if s["store"] else ()
        return _rotate(s["qkv"], s["positions"], s["inv_freq"], s["heads"], s["kv"], s["qw"], s["kw"], s["interleaved"], *cache)
    if s["kind"] == "pages":
        return _pages(s["table"], s["seen"], s["new"], s["free"], s["taken"], s["page"], s["tokens"])
    return _route(s["logits"], s["top_k"], s["scoring"], s["bias"], s["groups"], s["top_groups"], s["renormalize"], s["scale"])


def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "attend":
        lens = _spread(case["seqs"], case["low"], case["high"])
        read = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        h, kv, d = case["heads"], case["kv"], case["dim"]
        return {"bytes": read * kv * d * 2 * size + case["seqs"] * (2 * h * d * size + 4) + 4 * read // case["page"], "flops": 4 * read * h * d}
    if case["kind"] == "rotate":
        t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
        rows = 2 * h + (4 * kv if case["store"] else 2 * kv)
        return {"bytes": t * rows * d * size + t * (12 if case["store"] else 4), "flops": t * (h + kv) * d * 6}
    if case["kind"] == "pages":
        r, tokens = case["requests"], _tokens(case)
        return {"bytes": 16 * r + 12 * tokens + 8 * (tokens // case["page"]), "flops": tokens}
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    return {"bytes": t * e * size + t * k * 8 + (4 * e if case["bias"] else 0), "flops": 8 * t * e}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        kv, page, group = case["kv"], case["page"], case["heads"] // case["kv"]
        outs, norms = [], []
        for b, n in enumerate(s["lens"].tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            where = np.arange(first, n)
            names = s["table"][b].cpu().numpy().astype(np.int64)
            slot = torch.from_numpy(names[where // page] * page + where % page).to(s["q"].device)
            keys, values = (s[x].view(-1, kv, case["dim"]).index_select(0, slot).double() for x in ("k", "v"))
            score = torch.einsum("kgd,nkd->kgn", s["q"][b].double().view(kv, group, -1), keys) * s["scale"]
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            norm = torch.logsumexp(score, -1)
            outs.append(torch.einsum("kgn,nkd->kgd", torch.exp(score - norm[..., None]), values).reshape(case["heads"], -1))
            norms.append(norm.reshape(-1))
        o = torch.stack(outs)
        return (o, torch.stack(norms)) if case["lse"] else o
    if case["kind"] == "rotate":
        h, kv, d, half = case["heads"], case["kv"], case["dim"], case["rotated"] // 2
        x = s["qkv"].double().view(case["tokens"], h + 2 * kv, d)
        first = torch.arange(half, device=x.device) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        turn = torch.polar(torch.ones((case["tokens"], half), dtype=torch.float64, device=x.device),
                           torch.outer(s["positions"].double(), s["inv_freq"].double()))[:, None]

        def rotated(y, w):
            if w is not None:
                y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q, k = rotated(x[:, :h], s["qw"]), rotated(x[:, h:h + kv], s["kw"])
        if not case["store"]:
            return q, k
        kc, vc = (s[c].double().view(-1, kv, d).clone() for c in ("kc", "vc"))
        real = torch.nonzero(s["slots"] >= 0)[:, 0]
        kc.index_copy_(0, s["slots"][real], k[real])
        vc.index_copy_(0, s["slots"][real], x[real, h + kv:])
        return q, kc.view(s["kc"].shape), vc.view(s["vc"].shape)
    if case["kind"] == "pages":
        return None        # whole numbers: compared as they are
    x = s["logits"].double().cpu().numpy()
    p = 1 / (1 + np.exp(-x)) if case["scoring"] == "sigmoid" else np.exp(x - x.max(1, keepdims=True))
    if case["scoring"] == "softmax":
        p /= p.sum(1, keepdims=True)
    c = x if s["bias"] is None else p + s["bias"].double().cpu().numpy()
    t, groups = c.shape[0], case["groups"]
    if groups > 1:
        g = c.reshape(t, groups, -1)
        value = g.max(-1) if s["bias"] is None else np.sort(g, -1)[..., -2:].sum(-1)
        order = np.argsort(-value, 1, kind="stable")[:, case["top_groups"]:]
        g = g.copy()
        np.put_along_axis(g, order[:, :, None], -np.inf, 1)
        c = g.reshape(t, -1)
    ids = np.argsort(-c, 1, kind="stable")[:, :case["top_k"]]
    w = np.take_along_axis(p, ids, 1)
    if case["renormalize"]:
        w = w / w.sum(1, keepdims=True)
    return torch.from_numpy(w * case["scale"]), torch.from_numpy(ids.astype(np.int32))
