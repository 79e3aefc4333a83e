"""Workloads of the cached-decoding operators: the page plan of a key/value cache, the qkv rows' norm, multi-axis
rotary positions and cache append, attention over the paged cache, and the few-token product with 4-bit weights.

Each case runs one operator once, either in plain elementary torch operations (32-bit arithmetic, one rounding at the
end) or, with ``own`` set, through this package's entry points.  Page pools are laid out as the package's heads are:
[page][kv head][token in page][D].
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GOLDEN = 0.6180339887498949


def _b2q():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sam-3d-objects-ggml_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2q
    return b2q


def spread(n, lo, hi):
    """n whole numbers spread evenly over lo..hi, in an order that repeats nothing (a golden-ratio sequence)."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * GOLDEN) % 1.0)) for i in range(n)]


def lengths(case):
    """(tokens already cached, new tokens) of every request."""
    b = case["requests"]
    return spread(b, case["cached_min"], case["cached_max"]), spread(b, case["new_min"], case["new_max"])[::-1]


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One decoding step of a small serving batch: a new token per request, 16-token pages.  Latency only.
        {"name": "plan-decode-48", "op": "plan", "requests": 48, "cached_min": 20, "cached_max": 6000, "new_min": 1,
         "new_max": 1, "page": 16, "width": 512},
        # The plan of a large prefill wave with long prompts among short ones: the token map is most of the work.
        {"name": "plan-prefill-1000", "op": "plan", "requests": 1000, "cached_min": 0, "cached_max": 4000, "new_min": 1,
         "new_max": 1500, "page": 32, "width": 256},
        # The q, k and v of one decoding step, grouped heads, one position per token (all three axes alike).
        {"name": "rope-decode-24", "op": "rope", "tokens": 24, "q_heads": 24, "kv_heads": 8, "dim": 128, "type": "bf16",
         "page": 64, "axes": 3, "norm": False, "interleaved": False, "grid": 0},
        # Eight objects of 4096 voxel tokens and 4 pose tokens each, 16 heads of 64, per-head RMS norm, (x, y, z) axes.
        {"name": "rope-voxels-8x4100", "op": "rope", "tokens": 32800, "q_heads": 16, "kv_heads": 16, "dim": 64,
         "type": "f16", "page": 64, "axes": 3, "norm": True, "interleaved": True, "grid": 16},
        # A few short requests decoding with full heads of 64: latency.
        {"name": "attn-decode-3-short", "op": "attn", "requests": 3, "cached_min": 70, "cached_max": 900, "new_min": 1,
         "new_max": 1, "q_heads": 16, "kv_heads": 16, "dim": 64, "type": "f16", "page": 16, "window": 0, "sinks": 0},
        # A full serving batch, grouped heads, contexts up to 24k: the cache's bytes are the work.
        {"name": "attn-decode-64-long", "op": "attn", "requests": 64, "cached_min": 900, "cached_max": 24000,
         "new_min": 1, "new_max": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "page": 64, "window": 0,
         "sinks": 0},
        # One very long conversation: few rows, so the key axis has to be split.
        {"name": "attn-decode-1-120k", "op": "attn", "requests": 1, "cached_min": 120001, "cached_max": 120001,
         "new_min": 1, "new_max": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "f16", "page": 128, "window": 0,
         "sinks": 0},
        # Streaming: a window of 4096 keys and 4 first tokens that stay visible, odd group of 6, short drafts of tokens.
        {"name": "attn-stream-16-window", "op": "attn", "requests": 16, "cached_min": 3000, "cached_max": 30000,
         "new_min": 1, "new_max": 5, "q_heads": 24, "kv_heads": 4, "dim": 128, "type": "f16", "page": 32,
         "window": 4096, "sinks": 4},
        # Chunks of a long prompt over what is cached of it: tensor-core work.
        {"name": "attn-chunk-2x4096", "op": "attn", "requests": 2, "cached_min": 3000, "cached_max": 12000,
         "new_min": 3901, "new_max": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "page": 64,
         "window": 0, "sinks": 0},
        # The modulation projection of one sample (1024 -> 6 x 1024): the smallest product.
        {"name": "vec-q4_0-6144x1024-m1", "op": "vec", "n": 6144, "k": 1024, "m": 1, "type": "f32", "weights": "q4_0",
         "residual": False},
        # A branch's projection for four tokens, added to the residual stream.
        {"name": "vec-q4_0-8192x4096-m4", "op": "vec", "n": 8192, "k": 4096, "m": 4, "type": "f32", "weights": "q4_0",
         "residual": True},
        # A large projection for one token: the weight's bytes are the work.
        {"name": "vec-q4_k-49152x8192-m1", "op": "vec", "n": 49152, "k": 8192, "m": 1, "type": "bf16",
         "weights": "q4_k", "residual": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "vec", "vec"])
    if op == "plan":
        page = rng.choice([16, 32, 64, 128])
        requests = _log(rng, 1, 1000)
        hi = _log(rng, 1, 1500)
        cached = _log(rng, 1, 4000)
        return {"op": op, "requests": requests, "cached_min": 0, "cached_max": cached, "new_min": min(1, hi), "new_max": hi,
                "page": page, "width": (cached + hi) // page + rng.randint(1, 9)}
    if op == "rope":
        kv = rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 128])
        most = 32800 * 48 * 64 // (kv * (group + 2) * dim)
        return {"op": op, "tokens": _log(rng, 1, max(2, min(most, 40000))), "q_heads": kv * group, "kv_heads": kv,
                "dim": dim, "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
                "axes": rng.choice([1, 2, 3]), "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.5,
                "grid": rng.choice([0, 0, 16, 48])}
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 8])
        dim = rng.choice([64, 128])
        if rng.random() < 0.6:  # decoding: 1 to 6 new tokens
            new, requests = rng.choice([1, 1, 1, 2, 6]), _log(rng, 1, 64)
            cached = min(_log(rng, 1, 100000), 1500000 * 4 // (requests * max(kv, 4)))
        else:
            new, requests = _log(rng, 7, 2000), rng.randint(1, 4)
            cached = _log(rng, 1, 12000)
        windowed = rng.random() < 0.4
        return {"op": op, "requests": requests, "cached_min": cached // rng.randint(1, 20), "cached_max": cached,
                "new_min": max(1, new // 2), "new_max": new, "q_heads": kv * group, "kv_heads": kv, "dim": dim,
                "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
                "window": _log(rng, 1, 8000) if windowed else 0, "sinks": rng.randint(0, 70) if windowed else 0}
    weights = rng.choice(["q4_0", "q4_k"])
    k = 32 * _log(rng, 1, 512) if weights == "q4_0" else 256 * _log(rng, 1, 64)
    return {"op": op, "n": _log(rng, 1, min(60000, 400000000 // k)), "k": k, "m": rng.randint(1, 8),
            "type": rng.choice(["f32", "f16", "bf16"]), "weights": weights, "residual": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn, "vec": _prepare_vec}[case["op"]](case, g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _tables(cached, new, page, width, g):
    """Block table [B, width] of the cached and new tokens, pages in random order, -1 beyond; and the pool's size."""
    need = [_pages(c + n, page) for c, n in zip(cached, new)]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=g, device=DEV).int()
    table = torch.full((len(need), width), -1, dtype=torch.int32, device=DEV)
    col = torch.arange(width, device=DEV)[None, :]
    base = torch.cumsum(_ints(need), 0) - _ints(need)
    mask = col < _ints(need)[:, None]
    table[mask] = ids[(base[:, None] + col)[mask]]
    return table, pool


def _prepare_plan(case, g):
    cached, new = lengths(case)
    order = torch.randperm(len(cached), generator=g, device=DEV)
    cached_t, new_t = _ints(cached)[order], _ints(new)[order]
    page, width = case["page"], case["width"]
    table, used = _tables(cached_t.tolist(), [0] * len(cached), page, width, g)
    fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
    free = used + torch.randperm(fresh + 5, generator=g, device=DEV).int()
    return {"op": "plan", "cached": cached_t, "new": new_t, "page": page, "table": table, "free": free,
            "tokens": sum(new)}


def _prepare_rope(case, g):
    t, hq, hkv, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    dt = DTYPE[case["type"]]
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g, device=DEV) * 1.5
    i = torch.arange(t, device=DEV)
    axes, grid = case["axes"], case["grid"]
    if grid:  # voxel coordinates of a grid^3 volume, object after object
        coords = [i // (grid * grid) % grid, i // grid % grid, i % grid]
    else:  # running text: every axis counts the tokens, from a random start
        start = int(torch.randint(0, 5000, (1,), generator=g, device=DEV))
        coords = [i % 4096 + start] * 3
    pos = torch.stack(coords[:axes]).int()
    pairs = d // 2
    sections = [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)
    inv_freq = torch.exp(torch.arange(pairs, device=DEV, dtype=torch.float32) * (-math.log(10000.0) / pairs))
    n_pages = _pages(t, page) + 2
    slots = torch.randperm(n_pages * page, generator=g, device=DEV)[:t].contiguous()
    kc = torch.randn(n_pages, hkv, page, d, generator=g, device=DEV).to(dt)
    vc = torch.randn(n_pages, hkv, page, d, generator=g, device=DEV).to(dt)
    gq = gk = None
    if case["norm"]:
        gq = 1 + 0.2 * torch.randn(hq * d, generator=g, device=DEV)
        gk = 1 + 0.2 * torch.randn(hkv * d, generator=g, device=DEV)
    axis_of = torch.repeat_interleave(torch.arange(axes, device=DEV), _ints(sections, torch.int64))
    return {"op": "rope", "qkv": qkv, "hq": hq, "hkv": hkv, "d": d, "page": page, "pos": pos, "sections": sections,
            "axis_of": axis_of, "inv_freq": inv_freq, "slots": slots, "kc": kc, "vc": vc, "gq": gq, "gk": gk,
            "norm": case["norm"], "interleaved": case["interleaved"], "dt": dt}


def _prepare_attn(case, g):
    cached, new = lengths(case)
    hq, hkv, d, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    dt = DTYPE[case["type"]]
    total = [c + n for c, n in zip(cached, new)]
    width = max(_pages(x, page) for x in total)
    table, pool = _tables(cached, new, page, width, g)
    t = sum(new)
    q = (torch.randn(t, hq * d, generator=g, device=DEV) * 1.5).to(dt)
    kc = torch.randn(pool, hkv, page, d, generator=g, device=DEV, dtype=dt)
    vc = torch.randn(pool, hkv, page, d, generator=g, device=DEV, dtype=dt)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    row = torch.repeat_interleave(torch.arange(len(new), device=DEV), _ints(new, torch.int64))
    return {"op": "attn", "q": q, "kc": kc, "vc": vc, "table": table, "cu": _ints(cu), "kv_len": _ints(total),
            "new": _ints(new), "row": row, "max_q": max(new), "max_kv": max(total), "hq": hq, "hkv": hkv, "d": d,
            "page": page, "window": case["window"], "sinks": case["sinks"], "dt": dt}


def _blocks_q4_0(n, k, g):
    """GGUF Q4_0 rows: per 32 values an fp16 scale and 16 bytes of two 4-bit codes."""
    raw = torch.randint(0, 256, (n, k // 32, 18), dtype=torch.uint8, generator=g, device=DEV)
    d = (0.01 * (1 + torch.rand(n, k // 32, 1, generator=g, device=DEV))).half()
    raw[:, :, :2] = d.view(torch.uint8)
    return raw.view(n, -1)


def _blocks_q4_k(n, k, g):
    """GGUF Q4_K rows: per 256 values two fp16 factors, eight 6-bit scales and minima, 128 bytes of codes."""
    raw = torch.randint(0, 256, (n, k // 256, 144), dtype=torch.uint8, generator=g, device=DEV)
    d = (0.0003 * (1 + torch.rand(n, k // 256, 2, generator=g, device=DEV))).half()
    d[:, :, 1] *= 7
    raw[:, :, :4] = d.view(torch.uint8).view(n, k // 256, 4)
    return raw.view(n, -1)


def _prepare_vec(case, g):
    n, k, m = case["n"], case["k"], case["m"]
    raw = (_blocks_q4_0 if case["weights"] == "q4_0" else _blocks_q4_k)(n, k, g)
    s = {"op": "vec", "raw": raw, "n": n, "k": k, "m": m, "weights": case["weights"],
         "x": torch.randn(m, k, generator=g, device=DEV).to(DTYPE[case["type"]]),
         "bias": 0.1 * torch.randn(n, generator=g, device=DEV), "gate": None, "resid": None}
    if case["residual"]:
        s["gate"] = torch.randn(n, generator=g, device=DEV)
        s["resid"] = torch.randn(m, n, generator=g, device=DEV)
    if own:  # laid out once when the weights are loaded
        b2q = _b2q()
        s["packed"] = b2q.weight_pack_q4_0(raw, k) if case["weights"] == "q4_0" else b2q.weight_pack(b2q.TYPE_Q4_K, raw, k)
    return s


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn, "vec": _own_vec}[s["op"]](s)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "vec": _plain_vec}[s["op"]](s)


def _own_plan(s):
    slots, pos, cu, kv_len, counts = _b2q().kv_cache_plan(s["cached"], s["new"], s["page"], s["free"], s["table"],
                                                          s["tokens"])
    return {"table": s["table"], "slots": slots, "pos": pos, "cu": cu, "kv_len": kv_len, "counts": counts}


def _own_rope(s):
    q = _b2q().qkv_rope_cache(s["qkv"], s["hq"], s["hkv"], s["d"], s["pos"], s["sections"], s["inv_freq"], s["slots"],
                              s["kc"], s["vc"], norm=s["norm"], gamma_q=s["gq"], gamma_k=s["gk"],
                              interleaved=s["interleaved"])
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _own_attn(s):
    return _b2q().attention_paged(s["q"], s["kc"], s["vc"], s["table"], s["kv_len"], s["cu"], s["max_q"], s["max_kv"],
                                  s["hq"], window=s["window"], sinks=s["sinks"])


def _own_vec(s):
    b2q = _b2q()
    return b2q.mul_vec(b2q.TYPE_Q4_0 if s["weights"] == "q4_0" else b2q.TYPE_Q4_K, s["packed"], s["n"], s["k"], s["x"],
                       bias=s["bias"], gate=s["gate"], resid=s["resid"])


def _plain_plan(s):
    page, table, free = s["page"], s["table"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    width, n_tok = table.shape[1], s["tokens"]
    total = cached + new
    had, need = _pages(cached, page), _pages(total, page)
    base = torch.cumsum(need - had, 0) - (need - had)
    col = torch.arange(width, device=table.device)[None, :]
    idx = base[:, None] + col - had[:, None]
    fits = (col < need[:, None]) & (idx < free.numel())
    fresh = torch.where(fits, free[idx.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(col < had[:, None], table, fresh))
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    t = torch.arange(n_tok, device=table.device)
    r = torch.searchsorted(cu[1:], t, right=True)
    pos = cached[r] + t - cu[r]
    p = table[r, pos // page].long()
    slots = torch.where(p >= 0, p * page + pos % page, -1)
    counts = torch.stack([(need - had).sum(), (slots < 0).sum()])
    return {"table": table, "slots": slots, "pos": pos.int(), "cu": cu.int(), "kv_len": total.int(),
            "counts": counts.int()}


def _plain_rope(s):
    d, hq, hkv, page = s["d"], s["hq"], s["hkv"], s["page"]
    t = s["qkv"].shape[0]
    x = s["qkv"].view(t, hq + 2 * hkv, d)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    if s["norm"]:
        gamma = torch.cat([s["gq"], s["gk"]]).view(1, hq + hkv, d)
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * gamma
    angle = s["pos"].float()[s["axis_of"]].t() * s["inv_freq"]  # [t, d/2]
    c, sn = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if s["interleaved"]:
        a, b = qk[..., 0::2], qk[..., 1::2]
        out = torch.stack([a * c - b * sn, b * c + a * sn], -1).reshape(qk.shape)
    else:
        a, b = qk[..., :d // 2], qk[..., d // 2:]
        out = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    out = out.to(s["dt"])
    at, off = s["slots"] // page, s["slots"] % page
    s["kc"][at, :, off] = out[:, hq:]
    s["vc"][at, :, off] = v.to(s["dt"])
    return {"q": out[:, :hq].reshape(t, hq * d), "k_cache": s["kc"], "v_cache": s["vc"]}


def _plain_attn(s):
    d, hq, hkv, page = s["d"], s["hq"], s["hkv"], s["page"]
    b, width = s["table"].shape
    group, mq, mk = hq // hkv, s["max_q"], width * page
    dev = s["q"].device
    at = s["table"].clamp(min=0).long()
    k = s["kc"][at].transpose(1, 2).reshape(b, hkv, mk, d).float()
    v = s["vc"][at].transpose(1, 2).reshape(b, hkv, mk, d).float()
    t = torch.arange(s["q"].shape[0], device=dev)
    row, col = s["row"], t - s["cu"].long()[s["row"]]
    q = torch.zeros(b, mq, hkv, group, d, device=dev)
    q[row, col] = s["q"].view(-1, hkv, group, d).float()
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, group * mq, d)
    p = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    i = s["kv_len"][:, None, None] - s["new"][:, None, None] + torch.arange(mq, device=dev)[None, :, None]
    j = torch.arange(mk, device=dev)[None, None, :]
    see = (j <= i) & (j < s["kv_len"][:, None, None])
    if s["window"] > 0:
        see &= (j > i - s["window"]) | (j < s["sinks"])
    p.view(b, hkv, group, mq, mk).masked_fill_(~see[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.view(b, hkv, group, mq, d).permute(0, 3, 1, 2, 4)[row, col]
    return o.reshape(-1, hq * d).to(s["dt"])


def _dequantize(s):
    raw, n, k = s["raw"], s["n"], s["k"]
    if s["weights"] == "q4_0":
        blk = raw.view(n, k // 32, 18)
        d = blk[:, :, :2].contiguous().view(torch.float16).float()
        codes = torch.cat([blk[:, :, 2:] & 15, blk[:, :, 2:] >> 4], -1).float() - 8
        return (d * codes).view(n, k)
    blk = raw.view(n, k // 256, 144)
    d = blk[:, :, :2].contiguous().view(torch.float16).float()
    dmin = blk[:, :, 2:4].contiguous().view(torch.float16).float()
    p, q, r = blk[:, :, 4:8], blk[:, :, 8:12], blk[:, :, 12:16]
    sc = torch.cat([p & 63, (r & 15) | ((p >> 6) << 4)], -1).float()
    mn = torch.cat([q & 63, (r >> 4) | ((q >> 6) << 4)], -1).float()
    codes = blk[:, :, 16:].view(n, k // 256, 4, 1, 32)
    codes = torch.cat([codes & 15, codes >> 4], 3).view(n, k // 256, 8, 32).float()
    return ((d * sc)[..., None] * codes - (dmin * mn)[..., None]).view(n, k)


def _plain_vec(s):
    y = s["x"].float() @ _dequantize(s).t() + s["bias"]
    if s["resid"] is not None:
        y = s["resid"] + s["gate"] * y
    return y


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = lengths(case)
        page, b, t = case["page"], len(cached), sum(new)
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        cols = sum(case["width"] - _pages(c, page) for c in cached)
        return {"bytes": 8 * b + 4 * fresh + 4 * cols + 12 * t + 4 * (2 * b + 1) + 8, "flops": 4 * t + cols}
    if op == "rope":
        t, d, hq, hkv = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        values = t * (hq + 2 * hkv) * d
        return {"bytes": 6 * values + 4 * t * case["axes"] + 8 * t + 2 * d, "flops": (7 if case["norm"] else 3) * values}
    if op == "attn":
        cached, new = lengths(case)
        hq, hkv, d, w, sinks = case["q_heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"]
        pairs = keys = 0
        for c, n in zip(cached, new):
            lo = max(0, c - w + 1) if w else 0  # the first token's window begins here
            keys += (c + n - lo) + min(sinks, lo)
            if not w:
                pairs += n * c + n * (n + 1) // 2
            else:
                pairs += sum(min(w, p + 1) + min(sinks, max(0, p - w + 1)) for p in range(c, c + n))
        return {"bytes": 4 * keys * hkv * d + 4 * sum(new) * hq * d, "flops": 4 * pairs * hq * d}
    n, k, m = case["n"], case["k"], case["m"]
    w = n * (k // 32) * 18 if case["weights"] == "q4_0" else n * (k // 256) * 144
    size = 4 if case["type"] == "f32" else 2
    return {"bytes": w + size * m * k + 4 * n + 4 * m * n + (4 * n + 4 * m * n if case["residual"] else 0),
            "flops": 2 * n * k * m}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attn": _exact_attn, "vec": _exact_vec}[case["op"]](s)


def _exact_plan(s):
    """Request after request, page after page."""
    page, free = s["page"], s["free"].tolist()
    table, cached, new = s["table"].cpu().numpy().copy(), s["cached"].tolist(), s["new"].tolist()
    taken, slots, pos, cu = 0, [], [], [0]
    for b, (c, n) in enumerate(zip(cached, new)):
        first, last = _pages(c, page), _pages(c + n, page)
        table[b, first:] = -1
        for j in range(first, last):
            table[b, j] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(c, c + n):
            at = int(table[b, i // page])
            slots.append(at * page + i % page if at >= 0 else -1)
            pos.append(i)
        cu.append(cu[-1] + n)
    return {"table": torch.from_numpy(table), "slots": torch.tensor(slots, dtype=torch.int64),
            "pos": torch.tensor(pos, dtype=torch.int32), "cu": torch.tensor(cu, dtype=torch.int32),
            "kv_len": torch.tensor([c + n for c, n in zip(cached, new)], dtype=torch.int32),
            "counts": torch.tensor([taken, sum(x < 0 for x in slots)], dtype=torch.int32)}


def _exact_rope(s):
    d, hq, hkv, page = s["d"], s["hq"], s["hkv"], s["page"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    kc, vc = s["kc"].double(), s["vc"].double()
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                        s["pos"].double()[s["axis_of"]].t() * s["inv_freq"].double())

    def turned(h, gamma):
        if s["norm"]:
            h = h / torch.sqrt(h.square().sum(-1, keepdim=True) / d + 1e-6) * gamma.double().view(-1, d)
        if s["interleaved"]:
            z = torch.complex(h[..., 0::2], h[..., 1::2]) * phase[:, None]
            return torch.view_as_real(z).flatten(-2)
        z = torch.complex(h[..., :d // 2], h[..., d // 2:]) * phase[:, None]
        return torch.cat([z.real, z.imag], -1)

    q = turned(x[:, :hq], s["gq"])
    flat_k, flat_v = (c.transpose(1, 2).reshape(-1, hkv, d) for c in (kc, vc))
    flat_k[s["slots"]] = turned(x[:, hq:hq + hkv], s["gk"])
    flat_v[s["slots"]] = x[:, hq + hkv:]
    shape = (-1, page, hkv, d)
    return {"q": q.reshape(-1, hq * d), "k_cache": flat_k.view(shape).transpose(1, 2).contiguous(),
            "v_cache": flat_v.view(shape).transpose(1, 2).contiguous()}


def _exact_attn(s):
    """Request after request, kv head after kv head, over the keys in token order."""
    d, hq, hkv = s["d"], s["hq"], s["hkv"]
    group, out = hq // hkv, []
    for b, (length, n) in enumerate(zip(s["kv_len"].tolist(), s["new"].tolist())):
        first = int(s["cu"][b])
        pages = s["table"][b, :_pages(length, s["page"])].long()
        i = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None, :]
        hidden = j > i
        if s["window"] > 0:
            hidden = hidden | ((i - j >= s["window"]) & (j >= s["sinks"]))
        bias = torch.zeros(n, length, dtype=torch.float64, device=DEV).masked_fill(hidden, -math.inf)
        heads = []
        for h in range(hkv):
            k = s["kc"][pages, h].reshape(-1, d)[:length].double()
            v = s["vc"][pages, h].reshape(-1, d)[:length].double()
            for e in range(h * group, (h + 1) * group):
                q = s["q"][first:first + n, e * d:(e + 1) * d].double()
                heads.append(torch.softmax(q @ k.t() * d ** -0.5 + bias, -1) @ v)
        out.append(torch.cat(heads, 1))
    return torch.cat(out)


def _exact_vec(s):
    """Super-block after super-block of each row, in slabs of rows."""
    n, k, x = s["n"], s["k"], s["x"].double()
    y = torch.empty(s["m"], n, dtype=torch.float64, device=DEV)
    for r0 in range(0, n, 4096):
        raw = s["raw"][r0:r0 + 4096]
        rows = raw.shape[0]
        if s["weights"] == "q4_0":
            blk = raw.reshape(rows, k // 32, 18)
            d = (blk[..., 0].int() | (blk[..., 1].int() << 8)).short().view(torch.float16).double()
            w = torch.empty(rows, k // 32, 32, dtype=torch.float64, device=DEV)
            w[..., :16] = (blk[..., 2:] % 16).double() - 8
            w[..., 16:] = (blk[..., 2:] // 16).double() - 8
            w *= d[..., None]
        else:
            blk = raw.reshape(rows, k // 256, 144)
            d = (blk[..., 0].int() | (blk[..., 1].int() << 8)).short().view(torch.float16).double()
            dm = (blk[..., 2].int() | (blk[..., 3].int() << 8)).short().view(torch.float16).double()
            w = torch.empty(rows, k // 256, 256, dtype=torch.float64, device=DEV)
            for j in range(8):
                if j < 4:
                    sc, mn = blk[..., 4 + j] % 64, blk[..., 8 + j] % 64
                else:
                    sc = blk[..., 8 + j] % 16 + blk[..., j] // 64 * 16
                    mn = blk[..., 8 + j] // 16 + blk[..., 4 + j] // 64 * 16
                codes = blk[..., 16 + 32 * (j // 2):48 + 32 * (j // 2)]
                codes = codes // 16 if j % 2 else codes % 16
                w[..., 32 * j:32 * j + 32] = (d * sc)[..., None] * codes.double() - (dm * mn)[..., None]
        y[:, r0:r0 + rows] = x @ w.reshape(rows, k).t()
    y += s["bias"].double()
    if s["resid"] is not None:
        y = s["resid"].double() + s["gate"].double() * y
    return y
