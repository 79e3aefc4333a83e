"""Workloads of the operators around a step's linears whose weights go by row, and of the check of drafted tokens: the
router of an expert layer with its row plan, the experts' products, low-rank adapters of many requests beside a shared
projection, and the verification of drafted tokens against the target's probabilities.

Each case runs one operator once, either in plain elementary torch operations (32-bit arithmetic, 64-bit where a value
next to a border decides, one rounding at the end) or, with ``own`` set, through this package's entry points.  A slot is
one (token, choice) pair, token after token; a plan is the slots sorted by group (``order``) and where each group begins
(``offsets``).
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _b2q():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sam-3d-objects-ggml_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2q
    return b2q


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # The router of one decoding step: latency only.
        {"name": "route-decode-12", "op": "route", "tokens": 12, "experts": 64, "top": 6, "type": "f32",
         "scoring": "softmax", "renorm": True, "bias": False},
        # The router of a wave of prompts, many fine experts, a balancing bias on the choice, sigmoid weights.
        {"name": "route-prompts-20k", "op": "route", "tokens": 20471, "experts": 160, "top": 8, "type": "bf16",
         "scoring": "sigmoid", "renorm": True, "bias": True},
        # One token's experts, gate and up projections: few weights, far from a full device's worth of tiles.
        {"name": "experts-glu-decode-1", "op": "experts", "tokens": 1, "padding": 0, "experts": 64, "top": 6, "k": 2048,
         "n": 1408, "type": "f16", "weights": "f16", "glu": True, "out": "rows"},
        # A decoding batch: most experts get one or a few rows, so the weights' bytes are the work.
        {"name": "experts-glu-decode-40", "op": "experts", "tokens": 40, "padding": 0, "experts": 64, "top": 4, "k": 2048,
         "n": 1024, "type": "bf16", "weights": "bf16", "glu": True, "out": "rows"},
        # The way back with 4-bit weights, each token's choices weighted and added to the residual stream.
        {"name": "experts-down-q4-decode-24", "op": "experts", "tokens": 24, "padding": 0, "experts": 64, "top": 6,
         "k": 1408, "n": 2048, "type": "f16", "weights": "q4_0", "glu": False, "out": "f32"},
        # A wave of prompts through gate and up projections: tensor-core work, groups of very different sizes.
        {"name": "experts-glu-prompts-8192", "op": "experts", "tokens": 8192, "padding": 0, "experts": 32, "top": 4,
         "k": 2048, "n": 1408, "type": "bf16", "weights": "bf16", "glu": True, "out": "rows"},
        # An odd number of tokens, some of them padding, 4-bit weights, joined and rounded once.
        {"name": "experts-down-q4-prompts-3001", "op": "experts", "tokens": 3001, "padding": 77, "experts": 24, "top": 3,
         "k": 1408, "n": 2048, "type": "f16", "weights": "q4_0", "glu": False, "out": "same"},
        # A decoding batch whose requests bring adapters of their own, on a square projection.
        {"name": "adapters-decode-32", "op": "adapters", "requests": 32, "tokens_min": 1, "tokens_max": 1, "adapters": 24,
         "rank": 16, "k": 4096, "n": 4096, "type": "f16", "out": "f32"},
        # Prompts of a few tenants, rank 64: the rows' bytes are the work.
        {"name": "adapters-prompts-12", "op": "adapters", "requests": 12, "tokens_min": 150, "tokens_max": 1300,
         "adapters": 7, "rank": 64, "k": 4096, "n": 6144, "type": "bf16", "out": "f32"},
        # Short chunks, small rank, odd widths, some requests without an adapter.
        {"name": "adapters-chunks-29", "op": "adapters", "requests": 29, "tokens_min": 1, "tokens_max": 60, "adapters": 40,
         "rank": 8, "k": 1000, "n": 1233, "type": "f16", "out": "f16"},
        # A few requests with short drafts over a middling vocabulary: latency.
        {"name": "verify-4", "op": "verify", "requests": 4, "drafts_min": 1, "drafts_max": 4, "vocab": 32000,
         "type": "bf16", "draft_probs": True},
        # A serving batch with drafts of up to 7 tokens and a large vocabulary: one row of both models per request.
        {"name": "verify-96", "op": "verify", "requests": 96, "drafts_min": 0, "drafts_max": 7, "vocab": 151001,
         "type": "f32", "draft_probs": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "experts", "adapters", "adapters", "verify"])
    if op == "route":
        experts = _log(rng, 2, 512)
        return {"op": op, "tokens": _log(rng, 1, min(20000, 3200000 // experts)), "experts": experts,
                "top": rng.randint(1, min(16, experts)), "type": rng.choice(["f32", "f16", "bf16"]),
                "scoring": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.6, "bias": rng.random() < 0.4}
    if op == "experts":
        weights = rng.choice(["f16", "bf16", "q4_0"])
        glu = rng.random() < 0.5
        step = 32 if weights == "q4_0" else 8
        k, n = step * _log(rng, 64 // step, 4096 // step), _log(rng, 16, 2500)
        experts = min(_log(rng, 1, 128), max(1, 250000000 // (k * n * (1 + glu))))
        top = rng.randint(1, min(8, experts))
        most = int(1.8e11 / (k * n * (1 + glu) * top))
        tokens = _log(rng, 1, max(1, min(9000, most)))
        return {"op": op, "tokens": tokens, "padding": rng.choice([0, 0, min(tokens - 1, 9), tokens // 3]),
                "experts": experts, "top": top, "k": k, "n": n, "type": "f16" if weights == "q4_0" else weights,
                "weights": weights, "glu": glu, "out": "rows" if glu else rng.choice(["rows", "f32", "same"])}
    if op == "adapters":
        k, n = 8 * _log(rng, 4, 1024), _log(rng, 8, 8192)
        rank = 8 * rng.choice([1, 1, 2, 2, 4, 6, 8, 16])
        tokens = _log(rng, 1, max(1, min(8000, 33000000 // (k + n))))
        requests = rng.randint(1, min(64, tokens))
        each = max(1, tokens // requests)
        return {"op": op, "requests": requests, "tokens_min": 1 if rng.random() < 0.5 else each, "tokens_max": each,
                "adapters": min(_log(rng, 1, 64), max(1, 100000000 // (rank * (k + n)))), "rank": rank, "k": k, "n": n,
                "type": rng.choice(["f16", "bf16"]), "out": rng.choice(["f32", "same"])}
    vocab, low = _log(rng, 100, 200000), rng.randint(0, 3)
    return {"op": op, "requests": _log(rng, 1, min(100, 14000000 // vocab)), "drafts_min": low,
            "drafts_max": low + rng.randint(0, 4), "vocab": vocab, "type": rng.choice(["f32", "f16", "bf16"]),
            "draft_probs": rng.random() < 0.8}


def spread(count, lo, hi):
    """count whole numbers spread evenly over lo..hi, in an order that repeats nothing (a golden-ratio sequence)."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * 0.6180339887498949) % 1.0)) for i in range(count)]


def choices(case):
    """[tokens, top] experts of every token, all of a token's different; favourites differ by a factor of a few, so some
    groups are large and some empty.  Which expert is which is up to the seed (prepare renames them)."""
    rng = np.random.default_rng(case["tokens"] * 1000 + case["experts"])
    liking = 0.7 * rng.standard_normal(case["experts"])
    noise = rng.gumbel(size=(case["tokens"], case["experts"]))
    ids = np.argsort(-(noise + liking), axis=1, kind="stable")[:, :case["top"]].copy()
    if case["padding"]:
        ids[-case["padding"]:] = -1
    return ids


def adapter_rows(case):
    """(rows, adapter) of every request; about one request in eight has no adapter (-1) where there are many."""
    rows = spread(case["requests"], case["tokens_min"], case["tokens_max"])
    own_adapter = [(7 * i + 3) % case["adapters"] for i in range(case["requests"])]
    return rows, [-1 if i % 8 == 5 else a for i, a in enumerate(own_adapter)]


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"route": _prepare_route, "experts": _prepare_experts, "adapters": _prepare_adapters,
            "verify": _prepare_verify}[case["op"]](case, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _plan(ids, groups):
    """(order int32, offsets int32 [groups + 1]): the slots by group, in slot order inside one; those of no group last."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= groups), groups, flat)
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(groups + 1, device=key.device))
    return order.int(), offsets.int()


def _prepare_route(case, g):
    t, e = case["tokens"], case["experts"]
    logits = (1.5 * _randn(g, t, e) + 0.5 * _randn(g, e)).to(DTYPE[case["type"]])
    return {"op": "route", "logits": logits, "top": case["top"], "scoring": case["scoring"], "renorm": case["renorm"],
            "bias": 0.3 * _randn(g, e) if case["bias"] else None, "scale": 2.5 if case["scoring"] == "sigmoid" else 1.0}


def _blocks_q4_0(rows, k, g):
    """GGUF Q4_0 rows: per 32 values an fp16 scale and 16 bytes of two 4-bit codes."""
    raw = torch.randint(0, 256, (rows, k // 32, 18), dtype=torch.uint8, generator=g, device=DEV)
    d = (0.2 / math.sqrt(k) * (1 + torch.rand(rows, k // 32, 1, generator=g, device=DEV))).half()
    raw[:, :, :2] = d.view(torch.uint8)
    return raw.view(rows, -1)


def _prepare_experts(case, g):
    t, e, top, k, n = (case[x] for x in ("tokens", "experts", "top", "k", "n"))
    dt, rows = DTYPE[case["type"]], n * (1 + case["glu"])
    name = torch.randperm(e, generator=g, device=DEV)
    ids = torch.from_numpy(choices(case)).to(DEV)[torch.randperm(t, generator=g, device=DEV)]
    ids = torch.where(ids < 0, -1, name[ids.clamp(min=0)]).int()
    order, offsets = _plan(ids, e)
    per_row = top if case["out"] == "rows" else 1  # the way back starts from one row per slot
    x = _randn(g, t * top // per_row, k).to(dt)
    s = {"op": "experts", "x": x, "per_row": per_row, "ids": ids, "order": order, "offsets": offsets, "n": n, "k": k,
         "e": e, "glu": case["glu"], "out": case["out"], "weights": case["weights"], "dt": dt, "resid": None,
         "most": int((offsets[1:] - offsets[:-1]).max())}
    if case["weights"] == "q4_0":
        s["w"] = _blocks_q4_0(e * rows, k, g)
        if own:  # laid out once when the weights are loaded
            s["w"] = _b2q().weight_pack_q4_0(s["w"], k)
    else:
        s["w"] = torch.randn(e, rows, k, generator=g, device=DEV, dtype=dt) / math.sqrt(k)
    if case["out"] != "rows":
        share = torch.rand(t, top, generator=g, device=DEV) + 0.1
        s["share"] = share / share.sum(1, keepdim=True)
    if case["out"] == "f32":
        s["resid"] = _randn(g, t, n)
    return s


def _prepare_adapters(case, g):
    k, n, r, a = (case[x] for x in ("k", "n", "rank", "adapters"))
    dt = DTYPE[case["type"]]
    rows, mine = adapter_rows(case)
    ids = torch.repeat_interleave(torch.tensor(mine, device=DEV), torch.tensor(rows, device=DEV)).int()
    order, offsets = _plan(ids, a)
    t = sum(rows)
    out = DTYPE["f32"] if case["out"] == "f32" else dt
    return {"op": "adapters", "x": _randn(g, t, k).to(dt), "a": (_randn(g, a, r, k) / math.sqrt(k)).to(dt),
            "b": (0.3 / math.sqrt(r) * _randn(g, a, n, r)).to(dt), "scales": 0.5 + torch.rand(a, generator=g, device=DEV),
            "y": _randn(g, t, n).to(out), "ids": ids, "order": order, "offsets": offsets,
            "most": int((offsets[1:] - offsets[:-1]).max())}


def _prepare_verify(case, g):
    b, v, dt = case["requests"], case["vocab"], DTYPE[case["type"]]
    drafts = spread(b, case["drafts_min"], case["drafts_max"])
    d = sum(drafts)
    logits = 2.5 * _randn(g, d + b, v)
    target = torch.softmax(logits, -1)
    owner = torch.repeat_interleave(torch.arange(b, device=DEV), torch.tensor(drafts, device=DEV))
    at = torch.arange(d, device=DEV) + owner  # the target's row of a draft
    guess = torch.softmax(logits[at] + 0.7 * _randn(g, d, v), -1)
    race = -torch.log(torch.rand(d, v, generator=g, device=DEV).clamp(min=1e-30))
    tokens = (guess / race).argmax(-1) if d else torch.zeros(0, dtype=torch.int64, device=DEV)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(drafts)]), dtype=torch.int32, device=DEV)
    return {"op": "verify", "target": target.to(dt), "guess": guess.to(dt) if case["draft_probs"] else None,
            "tokens": tokens.int(), "cu": cu, "u": torch.rand(d, generator=g, device=DEV),
            "v": torch.rand(b, generator=g, device=DEV), "owner": owner, "most": max(drafts)}


# --------------------------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return {"route": _own_route, "experts": _own_experts, "adapters": _own_adapters, "verify": _own_verify}[s["op"]](s)
    return {"route": _plain_route, "experts": _plain_experts, "adapters": _plain_adapters,
            "verify": _plain_verify}[s["op"]](s)


def _own_route(s):
    ids, weights, order, offsets = _b2q().moe_route(s["logits"], s["top"], bias=s["bias"], scoring=s["scoring"],
                                                    renorm=s["renorm"], scale=s["scale"])
    return {"ids": ids, "weights": weights, "order": order, "offsets": offsets}


def _own_experts(s):
    b2q = _b2q()
    wtype = {"f16": b2q.TYPE_F16, "bf16": b2q.TYPE_BF16, "q4_0": b2q.TYPE_Q4_0}[s["weights"]]
    # (rows that are joined stay fp32 until then: the joined ones are rounded, once)
    y = b2q.mul_mat_id(wtype, s["w"], s["n"], s["k"], s["x"], s["order"], s["offsets"], per_row=s["per_row"],
                       glu=s["glu"], out_dtype=None if s["out"] == "rows" else torch.float32)
    if s["out"] == "rows":
        return y
    return b2q.moe_combine(y, s["share"], s["ids"], resid=s["resid"], out_dtype=torch.float32 if s["out"] == "f32" else s["dt"])


def _own_adapters(s):
    # fp32 rows are updated where they are, as the plain form updates them
    return _b2q().lora_add(s["y"], s["x"], s["a"], s["b"], s["scales"], s["order"], s["offsets"],
                           out=s["y"] if s["y"].dtype is torch.float32 else None)


def _own_verify(s):
    accepted, tokens = _b2q().draft_verify(s["target"], s["guess"], s["tokens"], s["cu"], s["u"], s["v"])
    return {"accepted": accepted, "tokens": tokens}


def _plain_route(s):
    x = s["logits"].float()
    key = x if s["bias"] is None else x + s["bias"]
    key = torch.where(torch.isnan(key), -math.inf, key)
    key, at = torch.sort(key, dim=1, descending=True, stable=True)
    key, at = key[:, :s["top"]], at[:, :s["top"]]
    picked = x.gather(1, at)
    if s["scoring"] == "sigmoid":
        weights = 1 / (1 + torch.exp(-picked))
    else:
        weights = torch.exp(picked - x.amax(1, keepdim=True))
        weights = weights / torch.exp(x - x.amax(1, keepdim=True)).sum(1, keepdim=True)
    none = key == -math.inf
    weights = torch.where(none, 0.0, weights)
    if s["renorm"]:
        weights = weights / weights.sum(1, keepdim=True)
    ids = torch.where(none, -1, at).int()
    order, offsets = _plan(ids, x.shape[1])
    return {"ids": ids, "weights": weights * s["scale"], "order": order, "offsets": offsets}


def _dequantize(raw, rows, k):
    blk = raw.view(rows, k // 32, 18)
    d = blk[:, :, :2].contiguous().view(torch.float16).float()
    codes = torch.cat([blk[:, :, 2:] & 15, blk[:, :, 2:] >> 4], -1).float() - 8
    return (d * codes).view(rows, k)


def _padded(s, x, groups):
    """Where each sorted slot sits in [groups, most] (its group, its place there), of slots that have a group."""
    offsets, order = s["offsets"].long(), s["order"].long()
    sorted_at = torch.arange(order.numel(), device=x.device)
    group = torch.searchsorted(offsets[1:], sorted_at, right=True)
    there = group < groups
    group = group.clamp(max=groups - 1)
    return order, group, (sorted_at - offsets[group]).clamp(max=s["most"] - 1), there


def _plain_experts(s):
    n, k, e = s["n"], s["k"], s["e"]
    rows = n * (1 + s["glu"])
    w = _dequantize(s["w"], e * rows, k).view(e, rows, k) if s["weights"] == "q4_0" else s["w"].float()
    order, group, place, there = _padded(s, s["x"], e)
    # (slots of no group are sent to a place of their own, behind the groups')
    at = torch.where(there, group * s["most"] + place, e * s["most"])
    x = torch.zeros(e * s["most"] + 1, k, device=DEV)
    x[at] = s["x"].float()[order // s["per_row"]]
    y = torch.bmm(x[:-1].view(e, s["most"], k), w.transpose(1, 2)).view(-1, rows)
    if s["glu"]:
        y = y[:, :n] / (1 + torch.exp(-y[:, :n])) * y[:, n:]
    y = torch.cat([y, torch.zeros(1, n, device=DEV)])
    out = torch.empty(order.numel(), n, device=DEV)
    out[order] = y[at]
    if s["out"] == "rows":
        return out.to(s["dt"])
    share = torch.where(s["ids"] < 0, 0.0, s["share"])
    out = (out.view(*share.shape, n) * share[:, :, None]).sum(1)
    return out + s["resid"] if s["out"] == "f32" else out.to(s["dt"])


def _plain_adapters(s):
    groups, r, k = s["a"].shape
    order, group, place, there = _padded(s, s["x"], groups)
    at = torch.where(there, group * s["most"] + place, groups * s["most"])
    x = torch.zeros(groups * s["most"] + 1, k, device=DEV)
    x[at] = s["x"].float()[order]
    h = torch.bmm(x[:-1].view(groups, s["most"], k), s["a"].float().transpose(1, 2)) * s["scales"][:, None, None]
    d = torch.bmm(h, s["b"].float().transpose(1, 2)).flatten(0, 1)
    d = torch.cat([d, torch.zeros_like(d[:1])])
    y = s["y"].float()
    y[order] += d[at]
    return y.to(s["y"].dtype)


def _plain_verify(s):
    target, guess, tokens, cu = s["target"], s["guess"], s["tokens"].long(), s["cu"].long()
    b, d = cu.numel() - 1, tokens.numel()
    req = torch.arange(b, device=DEV)
    row = torch.arange(d, device=DEV)
    pt = target[row + s["owner"], tokens].double()
    qt = guess[row, tokens].double() if guess is not None else torch.ones_like(pt)
    keep = torch.ones(b, s["most"] + 1, dtype=torch.bool, device=DEV)
    keep[s["owner"], row - cu[s["owner"]]] = s["u"].double() * qt < pt
    count = cu[1:] - cu[:-1]
    accepted = torch.minimum(torch.cumprod(keep.int(), 1).sum(1), count)
    rejected = accepted < count
    first = cu[:-1] + accepted
    p = target[first + req].double()
    weight = p
    if d:
        at = first.clamp(max=d - 1)
        if guess is not None:
            q = guess[at].double()
        else:
            q = torch.zeros_like(p)
            q[req, tokens[at]] = 1.0
        weight = torch.where(rejected[:, None], (p - q).clamp(min=0), p)
        weight = torch.where(weight.sum(1, keepdim=True) > 0, weight, p)
    edge = torch.cumsum(weight, 1)
    token = (edge <= s["v"].double()[:, None] * edge[:, -1:]).sum(1)
    place = torch.arange(weight.shape[1], device=DEV)
    token = torch.minimum(token, torch.where(weight > 0, place, -1).amax(1))
    out = torch.full((d + b,), -1, dtype=torch.int32, device=DEV)
    kept = row - cu[s["owner"]] < accepted[s["owner"]]
    out[row + s["owner"]] = torch.where(kept, tokens, -1).int()
    out[first + req] = token.int()
    return {"accepted": accepted.int(), "tokens": out}


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "route":
        t, e, top = case["tokens"], case["experts"], case["top"]
        return {"bytes": t * e * SIZE[case["type"]] + 12 * t * top + 4 * (e + 1) + (4 * e if case["bias"] else 0),
                "flops": 4 * t * e}
    if op == "experts":
        t, top, k, n = case["tokens"], case["top"], case["k"], case["n"]
        ids = choices(case)
        rows = n * (1 + case["glu"])
        used, slots = len(np.unique(ids[ids >= 0])), int((ids >= 0).sum())
        weights = used * rows * (k // 32 * 18 if case["weights"] == "q4_0" else 2 * k)
        read = 2 * k * (t - case["padding"] if case["out"] == "rows" else slots) + 4 * t * top + 4 * (case["experts"] + 1)
        if case["out"] == "rows":
            return {"bytes": weights + read + 2 * t * top * n, "flops": 2 * slots * rows * k}
        read += 8 * t * top + (4 * t * n if case["out"] == "f32" else 0)
        return {"bytes": weights + read + (4 if case["out"] == "f32" else 2) * t * n, "flops": 2 * slots * n * (k + 1)}
    if op == "adapters":
        rows, mine = adapter_rows(case)
        k, n, r = case["k"], case["n"], case["rank"]
        live = sum(x for x, a in zip(rows, mine) if a >= 0)
        used = len({a for a in mine if a >= 0})
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": 2 * live * k + 2 * used * r * (k + n) + 2 * out * sum(rows) * n + 4 * sum(rows) + 4 * used,
                "flops": 2 * live * r * (k + n) + live * n}
    # one row of the target's probabilities per request, one of the draft's where a draft was turned down (of these
    # inputs, about one draft in five)
    drafts = spread(case["requests"], case["drafts_min"], case["drafts_max"])
    down = sum(1 - 0.8 ** x for x in drafts) if case["draft_probs"] else 0
    size, v = SIZE[case["type"]], case["vocab"]
    return {"bytes": int((len(drafts) + down) * v * size) + sum(drafts) * (12 + 2 * size) + 12 * len(drafts),
            "flops": int((2 * len(drafts) + down) * v)}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "experts": _exact_experts, "adapters": _exact_adapters,
            "verify": _exact_verify}[case["op"]](s)


def _groups(s):
    """Group after group: its slots."""
    offsets, order = s["offsets"].tolist(), s["order"].long()
    for i, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            yield i, order[lo:hi]


def _exact_route(s):
    x = s["logits"].double().cpu().numpy()
    t, e = x.shape
    choice = s["logits"].float().cpu().numpy()
    if s["bias"] is not None:  # the choice is made between 32-bit numbers
        choice = choice + s["bias"].cpu().numpy()
    ids = np.argsort(-choice, axis=1, kind="stable")[:, :s["top"]]
    if s["scoring"] == "sigmoid":
        score = 1 / (1 + np.exp(-x))
    else:
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    weights = np.take_along_axis(score, ids, 1)
    if s["renorm"]:
        weights = weights / weights.sum(1, keepdims=True)
    flat = ids.reshape(-1)
    return {"ids": torch.from_numpy(ids.astype(np.int32)), "weights": torch.from_numpy(weights * s["scale"]),
            "order": torch.from_numpy(np.argsort(flat, kind="stable").astype(np.int32)),
            "offsets": torch.from_numpy(np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e))]).astype(np.int32))}


def _exact_experts(s):
    n, k = s["n"], s["k"]
    rows = n * (1 + s["glu"])
    y = torch.zeros(s["order"].numel(), n, dtype=torch.float64, device=DEV)
    for e, slots in _groups(s):
        if s["weights"] == "q4_0":
            blk = s["w"][e * rows:(e + 1) * rows].reshape(rows, k // 32, 18)
            d = (blk[..., 0].int() | (blk[..., 1].int() << 8)).short().view(torch.float16).double()
            w = torch.empty(rows, k // 32, 32, dtype=torch.float64, device=DEV)
            w[..., :16] = (blk[..., 2:] % 16).double() - 8
            w[..., 16:] = (blk[..., 2:] // 16).double() - 8
            w = (w * d[..., None]).view(rows, k)
        else:
            w = s["w"][e].double()
        z = s["x"][slots // s["per_row"]].double() @ w.t()
        y[slots] = z[:, :n] * torch.sigmoid(z[:, :n]) * z[:, n:] if s["glu"] else z
    if s["out"] == "rows":
        return y
    t, top = s["ids"].shape
    total = torch.zeros(t, n, dtype=torch.float64, device=DEV) if s["resid"] is None else s["resid"].double()
    for j in range(top):  # (a slot of no group is a row of zeros)
        total = total + s["share"][:, j, None].double() * y[j::top]
    return total


def _exact_adapters(s):
    y = s["y"].double()
    for i, rows in _groups(s):
        y[rows] += float(s["scales"][i]) * (s["x"][rows].double() @ s["a"][i].double().t() @ s["b"][i].double().t())
    return y


def _exact_verify(s):
    """Request after request, draft after draft."""
    cu, tokens = s["cu"].tolist(), s["tokens"].tolist()
    u, v = s["u"].tolist(), s["v"].tolist()
    accepted, out = [], []
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        weight, new = None, []
        for i in range(lo, hi):
            p = s["target"][i + b].double()
            q = torch.zeros_like(p)
            if s["guess"] is None:
                q[tokens[i]] = 1.0
            else:
                q = s["guess"][i].double()
            if u[i] * float(q[tokens[i]]) < float(p[tokens[i]]):
                new.append(tokens[i])
                continue
            weight = (p - q).clamp(min=0)
            if float(weight.sum()) == 0:
                weight = p
            break
        if weight is None:
            weight = s["target"][hi + b].double()
        edge = weight.cpu().numpy().cumsum()
        token = int(np.searchsorted(edge, v[b] * edge[-1], side="right"))
        accepted.append(len(new))
        out += new + [min(token, int(np.flatnonzero(weight.cpu().numpy()).max()))] + [-1] * (hi - lo - len(new))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(out, dtype=torch.int32)}
