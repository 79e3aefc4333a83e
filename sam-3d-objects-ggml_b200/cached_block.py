"""A transformer block over a paged key / value cache, composed from libb2q's
cached-decoding entry points: what a graph that adds tokens to requests step by
step (a prompt's chunks, then single tokens) runs per layer.

    h = norm(x)                                        b2q_norm_modulate
    qkv = h . W_qkv + b_qkv                            b2q_mul_vec, or the Q4_0 GEMM
    q, k turned by their (x, y, z) positions after a   b2q_qkv_rope_cache
      per-head RMS norm; k, v into the cache
    o = softmax(q k^T / sqrt(D)) v over the cache      b2q_attention_paged
    x = x + (o . W_out + b_out)                        b2q_mul_vec, or the Q4_0 GEMM
    x = x + (gelu(norm(x) . W1 + b1) . W2 + b2)        same, with b2q_gelu between

Up to `unrounded_rows` rows (MUL_VEC_MAX_M unless the block is told more) the
linears are b2q_mul_vec's, eight rows at a time: the 4-bit weight's values
against unrounded activations.  More rows go to the tensor-core GEMM on the same
compact Q4_0 weights, which rounds the activations to Q8_0 as ggml's CPU mul_mat
does: a token's result depends, by that rounding, on which side of the number its
step is.

With `Experts` the last line is a mixture layer instead:

    choice, shares, rows by expert = route(h . W_r)    b2q_mul_mat_f32, b2q_moe_route
    z = silu(h . W_gate) * (h . W_up), per slot        b2q_mul_mat_id
    x = x + sum of shares * (z . W_down)               b2q_mul_mat_id, b2q_moe_combine

and with `Adapters` each linear that has some adds its row's low-rank product
(b2q_lora_add), the rows sorted by adapter once per step (b2q_group_rows); beside
experts those are qkv and out.

`PagedCache` keeps the pools, the block tables and the free pages of a set of
requests, and takes back the pages of those that end; the host knows the lengths
it asked for, the device builds the rest (b2q_kv_cache_plan), so a step never
waits for the device.  A step of drafted tokens ends with b2q_draft_verify, and
`keep` takes back what the turned down ones had; the lengths to keep are host
numbers, so whoever drafts reads the accepted counts back first, and waits for
that step.

    python cached_block.py       # a prompt of 300 tokens, then 8 single tokens
"""
from __future__ import annotations

import b2q


class PagedCache:
    """Pools [pages][kv heads][page size][D] of every layer, and who owns which page."""

    def __init__(self, dev, layers: int, requests: int, kv_heads: int, D: int, pages: int, page_size: int = 64,
                 max_len: int = 4096, dtype=None):
        import torch
        dtype = torch.float16 if dtype is None else dtype
        shape = (pages, kv_heads, page_size, D)
        self.k = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(layers)]
        self.page_size, self.dev = page_size, dev
        self.table = torch.full((requests, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)  # entries `taken` and on are the free pages
        self.taken = 0
        self.lengths = [0] * requests

    def plan(self, new: list, stream=None) -> dict:
        """Room for new[b] tokens of every request b; the step's slots, positions and lengths.  A step that
        runs on a given stream is planned on it too (the table and the free list are never reallocated)."""
        import torch
        with torch.cuda.stream(stream):
            return self._plan(new)

    def _plan(self, new: list) -> dict:
        import torch
        ps = self.page_size
        if min(new) < 0:
            raise ValueError("a step adds tokens")
        pages = sum(-(-(c + n) // ps) - -(-c // ps) for c, n in zip(self.lengths, new))
        if pages > self.free.numel() - self.taken or max(c + n for c, n in zip(self.lengths, new)) > self.table.shape[1] * ps:
            raise RuntimeError("the cache is full")
        # (from pinned memory: a copy from pageable memory would wait for all that the stream has to do)
        counts = torch.tensor([self.lengths, new], dtype=torch.int32).pin_memory().to(self.dev, non_blocking=True)
        slots, pos, cu, kv_len, _ = b2q.kv_cache_plan(counts[0], counts[1], ps, self.free[self.taken:], self.table, sum(new))
        self.taken += pages
        self.lengths = [c + n for c, n in zip(self.lengths, new)]
        return {"slots": slots, "pos": pos, "cu": cu, "kv_len": kv_len, "max_new": max(new), "max_kv": max(self.lengths)}

    def release(self, request: int, stream=None) -> None:
        """Ends a request: its pages are free again, and its number is there for another one."""
        import torch
        with torch.cuda.stream(stream):
            pages = -(-self.lengths[request] // self.page_size)
            self.free[self.taken - pages:self.taken].copy_(self.table[request, :pages])
            self.table[request].fill_(-1)
        self.taken -= pages
        self.lengths[request] = 0

    def keep(self, request: int, length: int, stream=None) -> None:
        """Takes a request back to its first `length` tokens (drafts that were turned down): the pages behind them
        are free again."""
        import torch
        ps, old = self.page_size, self.lengths[request]
        if not 0 <= length <= old:
            raise ValueError("a request keeps some of its tokens")
        first, last = -(-length // ps), -(-old // ps)
        if last > first:
            with torch.cuda.stream(stream):
                self.free[self.taken - (last - first):self.taken].copy_(self.table[request, first:last])
                self.table[request, first:last].fill_(-1)
        self.taken -= last - first
        self.lengths[request] = length


def fp16_rows(x):
    """(fp16 rows, powers of two fp32 [rows]) whose products are the rows of x, up to the rounding of fp16: a row whose
    values pass fp16's range is divided by its power of two, for all others that is 1."""
    import torch
    top = x.abs().amax(1).float()
    exponent = torch.frexp(top).exponent
    above = torch.where(torch.isfinite(top), exponent - 15, 0).clamp(min=0).int()
    power = ((above + 127) << 23).view(torch.float32)
    return (x / power[:, None]).half(), power


class Experts:
    """A mixture layer's weights: the router's rows fp32 [E, C]; every expert's gate and up rows (2 * hidden of C) and
    rows of the way back (C of hidden) as GGUF Q4_0 rows, one expert under another.  bias (fp32 [E]) is the router's
    correction bias: it is added to the scores for the choice, and never enters the shares; bias_on="logit" adds it
    to the logits instead."""

    def __init__(self, dev, router, w_in, w_out, C: int, hidden: int, top: int, scoring: str = "softmax", renorm: bool = True,
                 scale: float = 1.0, bias=None, bias_on: str = "score"):
        import torch
        self.router, self.C, self.hidden, self.top, self.bias = router, C, hidden, top, bias
        self.how = {"scoring": scoring, "renorm": renorm, "scale": scale, "bias_on": bias_on}
        raw = torch.from_numpy(w_in).to(dev)
        self.hidden_fits_fp16 = self.hidden_bound(raw, C, hidden) <= 65504 * (1 - 2.0 ** -8)
        self.w_in = b2q.weight_pack_q4_0(raw, C)
        self.w_out = b2q.weight_pack_q4_0(torch.from_numpy(w_out).to(dev), hidden)

    @staticmethod
    def hidden_bound(raw, C: int, hidden: int) -> float:
        """What |silu(gate) * up| cannot pass for normed rows (no longer than sqrt(C)): C |gate row| |up row|, the largest."""
        import torch
        worst = 0.0
        for rows in raw.view(-1, 2 * hidden, C // 32, 18):  # an expert at a time
            d = rows[:, :, :2].contiguous().view(torch.float16)[:, :, 0].double()
            codes = torch.cat([rows[:, :, 2:] & 15, rows[:, :, 2:] >> 4], -1).to(torch.int16) - 8
            length = (d.square() * codes.square().sum(-1)).sum(-1).sqrt()
            bound = float((C * length[:hidden] * length[hidden:]).max())
            worst = max(worst, bound) if bound == bound else float("inf")
        return worst

    def forward(self, h, x):
        """x += the layer's output for the normed rows h (fp32 [tokens, C], no longer than sqrt(C)), in place.  The rows of
        both products are fp16; hidden values that the weights let pass its range (hidden_bound) are taken by a
        power of two per row, which their shares give back."""
        import torch
        logits = b2q.mul_mat_f32(self.router, h)
        ids, shares, order, offsets = b2q.moe_route(logits, self.top, bias=self.bias, **self.how)
        z = b2q.mul_mat_id(b2q.TYPE_Q4_0, self.w_in, self.hidden, self.C, h.half(), order, offsets, per_row=self.top, glu=True,
                           out_dtype=None if self.hidden_fits_fp16 else torch.float32)
        if not self.hidden_fits_fp16:
            z, power = fp16_rows(z)
            shares = shares * power.view_as(shares)
        y = b2q.mul_mat_id(b2q.TYPE_Q4_0, self.w_out, self.C, self.hidden, z, order, offsets, out_dtype=torch.float32)
        return b2q.moe_combine(y, shares, ids, resid=x, out=x)


class Adapters:
    """Low-rank adapters of a block's linears: {"qkv" | "out" | "fc1" | "fc2": (a [G, rank, in], b [G, out, rank])} in fp16,
    and their scales fp32 [G] (or None).  A block with experts has no fc1 and fc2 and refuses adapters for them."""

    def __init__(self, pairs: dict, scales=None):
        if not pairs or not set(pairs) <= {"qkv", "out", "fc1", "fc2"}:
            raise ValueError("adapters belong to qkv, out, fc1 or fc2")
        self.pairs, self.scales = pairs, scales
        self.count = next(iter(pairs.values()))[0].shape[0]

    def plan(self, ids, stream=None):
        """A step's rows by adapter, for every layer's pass: ids int32 [tokens], -1 for none."""
        return b2q.group_rows(ids, self.count, stream=stream)

    def add(self, name: str, y, x, rows):
        """y (fp32) += the adapters' products of the rows x, in place.  The rows are taken as fp16: normed ones (qkv, fc1)
        and those of an fp16 cache (out) lie in its range, others are divided by a power of two that comes back."""
        import torch
        if name in self.pairs:
            a, b = self.pairs[name]
            power = None
            if name in ("qkv", "fc1") or x.dtype is torch.float16:
                x = x.half()
            else:
                x, power = fp16_rows(x)
            b2q.lora_add(y, x, a, b, self.scales, *rows, out=y, row_scales=power)
        return y


class CachedBlock:
    """One block's Q4_0 weights and its forward pass on fp32 rows x [tokens, C]."""

    @staticmethod
    def shapes(C: int, heads: int, kv_heads: int, D: int, hidden: int) -> dict:
        return {"qkv": ((heads + 2 * kv_heads) * D, C), "out": (C, heads * D), "fc1": (hidden, C), "fc2": (C, hidden)}

    def __init__(self, dev, weights: dict, vectors: dict, C: int, heads: int, kv_heads: int, D: int, hidden: int,
                 sections, inv_freq, window: int = 0, sinks: int = 0, unrounded_rows: int = b2q.MUL_VEC_MAX_M,
                 experts: Experts | None = None):
        """weights: GGUF Q4_0 rows (uint8 numpy [out, row bytes]); vectors: fp32 device tensors
        b_qkv, b_out, b1, b2 and the RMS gammas gq [heads * D], gk [kv_heads * D].  Steps of up to
        unrounded_rows tokens keep the activations of the linears as they are, more round them to Q8_0.
        With experts, fc1 and fc2 (and their biases) are not used and may be absent."""
        import torch
        self.unrounded_rows, self.experts = unrounded_rows, experts
        self.C, self.H, self.Hk, self.D, self.hidden = C, heads, kv_heads, D, hidden
        self.sections, self.inv_freq, self.window, self.sinks = tuple(sections), inv_freq, window, sinks
        self.shape = self.shapes(C, heads, kv_heads, D, hidden)
        self.packed = {n: b2q.weight_pack_q4_0(torch.from_numpy(weights[n]).to(dev), k) for n, (_, k) in self.shape.items()
                       if experts is None or n in ("qkv", "out")}
        self.vec = vectors

    def _linear(self, name: str, x, bias, resid=None):
        n, k = self.shape[name]
        m = x.shape[0]
        if m <= min(self.unrounded_rows, b2q.MUL_VEC_MAX_M):
            return b2q.mul_vec(b2q.TYPE_Q4_0, self.packed[name], n, k, x, bias=bias, resid=resid, out=resid)
        if m <= self.unrounded_rows:
            import torch
            y = resid if resid is not None else torch.empty((m, n), dtype=torch.float32, device=x.device)
            for i in range(0, m, b2q.MUL_VEC_MAX_M):
                part = slice(i, i + b2q.MUL_VEC_MAX_M)
                b2q.mul_vec(b2q.TYPE_Q4_0, self.packed[name], n, k, x[part], bias=bias,
                            resid=None if resid is None else resid[part], out=y[part])
            return y
        act = b2q.act_prepare(x.float())
        return b2q.mul_mat_prepared_q4_0(self.packed[name], n, k, act, m, bias=bias, resid=resid, out=resid)

    def forward(self, x, cache: PagedCache, layer: int, step: dict, positions, stream=None, adapters: Adapters | None = None,
                rows=None):
        """x: fp32 [tokens, C], updated in place and returned; positions int32 [axes, tokens].  With a stream the
        whole pass belongs to it: its casts, and the pool that its temporaries come from and go back to.
        adapters: this layer's, with rows = adapters.plan(...) of the step."""
        import torch
        if self.experts is not None and adapters is not None and ("fc1" in adapters.pairs or "fc2" in adapters.pairs):
            raise ValueError("adapters for fc1 or fc2, whose place the experts have taken")
        with torch.cuda.stream(stream):
            return self._forward(x, cache, layer, step, positions, adapters, rows)

    def _forward(self, x, cache: PagedCache, layer: int, step: dict, positions, adapters, rows):
        v = self.vec
        add = (lambda name, y, inp: adapters.add(name, y, inp, rows)) if adapters is not None else (lambda name, y, inp: y)
        h = b2q.norm_modulate(x)
        qkv = add("qkv", self._linear("qkv", h, v["b_qkv"]), h)
        k, vv = cache.k[layer], cache.v[layer]
        q = b2q.qkv_rope_cache(qkv, self.H, self.Hk, self.D, positions, self.sections, self.inv_freq, step["slots"], k, vv,
                               norm=True, gamma_q=v["gq"], gamma_k=v["gk"])
        o = b2q.attention_paged(q, k, vv, cache.table, step["kv_len"], step["cu"], step["max_new"], step["max_kv"], self.H,
                                window=self.window, sinks=self.sinks)
        add("out", self._linear("out", o, v["b_out"], resid=x), o)
        h = b2q.norm_modulate(x)
        if self.experts is not None:
            return self.experts.forward(h, x)
        h = b2q.gelu(add("fc1", self._linear("fc1", h, v["b1"]), h))
        add("fc2", self._linear("fc2", h, v["b2"], resid=x), h)
        return x


def random_q4_0(rng, n: int, k: int):
    """Seeded GGUF Q4_0 rows of random codes (uint8 numpy [n, row bytes])."""
    import numpy as np
    raw = rng.integers(0, 256, (n, k // 32, 18), dtype=np.uint8)
    d = (rng.uniform(0.5, 1.0, (n, k // 32, 1)) * 0.3 / k ** 0.5).astype(np.float16)
    raw[:, :, :2] = d.view(np.uint8)
    return raw.reshape(n, -1)


def random_experts(dev, E: int, C: int, hidden: int, top: int, seed: int = 0, **kw):
    """A mixture layer with seeded weights, and its raw rows (router, gate and up, down)."""
    import numpy as np
    import torch
    rng = np.random.default_rng(seed)
    router = (rng.standard_normal((E, C)) / C ** 0.5).astype(np.float32)
    w_in, w_out = random_q4_0(rng, E * 2 * hidden, C), random_q4_0(rng, E * C, hidden)
    return Experts(dev, torch.from_numpy(router).to(dev), w_in, w_out, C, hidden, top, **kw), (router, w_in, w_out)


def random_block(dev, C: int, heads: int, kv_heads: int, D: int, hidden: int, sections, seed: int = 0, **kw):
    """A block with seeded weights (Q4_0 blocks of random codes), and its raw rows."""
    import numpy as np
    import torch
    rng = np.random.default_rng(seed)
    weights = {}
    for name, (n, k) in CachedBlock.shapes(C, heads, kv_heads, D, hidden).items():
        weights[name] = random_q4_0(rng, n, k)
    f = lambda n, mean, s: torch.from_numpy((mean + s * rng.standard_normal(n)).astype(np.float32)).to(dev)  # noqa: E731
    vec = {"b_qkv": f((heads + 2 * kv_heads) * D, 0, 0.1), "b_out": f(C, 0, 0.1), "b1": f(hidden, 0, 0.1),
           "b2": f(C, 0, 0.1), "gq": f(heads * D, 1, 0.1), "gk": f(kv_heads * D, 1, 0.1)}
    pairs = sum(sections)
    inv_freq = torch.from_numpy((100.0 ** (-np.arange(pairs) / pairs)).astype(np.float32)).to(dev)
    return CachedBlock(dev, weights, vec, C, heads, kv_heads, D, hidden, sections, inv_freq, **kw), weights


def main():
    import torch
    dev = torch.device("cuda", torch.cuda.current_device())
    C, heads, D = 1024, 16, 64
    block, _ = random_block(dev, C, heads, heads, D, 4 * C, (12, 10, 10))
    cache = PagedCache(dev, 1, 1, heads, D, pages=16)
    x = torch.randn(308, C, device=dev)
    for lo, hi in [(0, 300)] + [(t, t + 1) for t in range(300, 308)]:
        step = cache.plan([hi - lo])
        p = step["pos"]
        grid = torch.stack([p // 64, p // 8 % 8, p % 8]).int()  # an 8 x 8 x n volume, voxel after voxel
        y = block.forward(x[lo:hi].clone(), cache, 0, step, grid)
        print(f"tokens {lo}..{hi - 1}: output rms {float(y.square().mean().sqrt()):.4f}, cached {cache.lengths[0]}")
    status = b2q.device_status()
    if status:
        raise SystemExit(f"device status 0x{status:x}")


if __name__ == "__main__":
    main()
