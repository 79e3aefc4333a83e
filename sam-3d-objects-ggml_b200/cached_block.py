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

`PagedCache` keeps the pools, the block tables and the free pages of a set of
requests, and takes back the pages of those that end; the host knows the lengths
it asked for, the device builds the rest (b2q_kv_cache_plan), so a step never
waits for the device.

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


class CachedBlock:
    """One block's Q4_0 weights and its forward pass on fp32 rows x [tokens, C]."""

    @staticmethod
    def shapes(C: int, heads: int, kv_heads: int, D: int, hidden: int) -> dict:
        return {"qkv": ((heads + 2 * kv_heads) * D, C), "out": (C, heads * D), "fc1": (hidden, C), "fc2": (C, hidden)}

    def __init__(self, dev, weights: dict, vectors: dict, C: int, heads: int, kv_heads: int, D: int, hidden: int,
                 sections, inv_freq, window: int = 0, sinks: int = 0, unrounded_rows: int = b2q.MUL_VEC_MAX_M):
        """weights: GGUF Q4_0 rows (uint8 numpy [out, row bytes]); vectors: fp32 device tensors
        b_qkv, b_out, b1, b2 and the RMS gammas gq [heads * D], gk [kv_heads * D].  Steps of up to
        unrounded_rows tokens keep the activations of the linears as they are, more round them to Q8_0."""
        import torch
        self.unrounded_rows = unrounded_rows
        self.C, self.H, self.Hk, self.D, self.hidden = C, heads, kv_heads, D, hidden
        self.sections, self.inv_freq, self.window, self.sinks = tuple(sections), inv_freq, window, sinks
        self.shape = self.shapes(C, heads, kv_heads, D, hidden)
        self.packed = {n: b2q.weight_pack_q4_0(torch.from_numpy(weights[n]).to(dev), k) for n, (_, k) in self.shape.items()}
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

    def forward(self, x, cache: PagedCache, layer: int, step: dict, positions, stream=None):
        """x: fp32 [tokens, C], updated in place and returned; positions int32 [axes, tokens].  With a stream the
        whole pass belongs to it: its casts, and the pool that its temporaries come from and go back to."""
        import torch
        with torch.cuda.stream(stream):
            return self._forward(x, cache, layer, step, positions)

    def _forward(self, x, cache: PagedCache, layer: int, step: dict, positions):
        v = self.vec
        h = b2q.norm_modulate(x)
        qkv = self._linear("qkv", h, v["b_qkv"])
        k, vv = cache.k[layer], cache.v[layer]
        q = b2q.qkv_rope_cache(qkv, self.H, self.Hk, self.D, positions, self.sections, self.inv_freq, step["slots"], k, vv,
                               norm=True, gamma_q=v["gq"], gamma_k=v["gk"])
        o = b2q.attention_paged(q, k, vv, cache.table, step["kv_len"], step["cu"], step["max_new"], step["max_kv"], self.H,
                                window=self.window, sinks=self.sinks)
        self._linear("out", o, v["b_out"], resid=x)
        h = b2q.gelu(self._linear("fc1", b2q.norm_modulate(x), v["b1"]))
        self._linear("fc2", h, v["b2"], resid=x)
        return x


def random_block(dev, C: int, heads: int, kv_heads: int, D: int, hidden: int, sections, seed: int = 0, **kw):
    """A block with seeded weights (Q4_0 blocks of random codes), and its raw rows."""
    import numpy as np
    import torch
    rng = np.random.default_rng(seed)
    weights = {}
    for name, (n, k) in CachedBlock.shapes(C, heads, kv_heads, D, hidden).items():
        raw = rng.integers(0, 256, (n, k // 32, 18), dtype=np.uint8)
        d = (rng.uniform(0.5, 1.0, (n, k // 32, 1)) * 0.3 / k ** 0.5).astype(np.float16)
        raw[:, :, :2] = d.view(np.uint8)
        weights[name] = raw.reshape(n, -1)
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
