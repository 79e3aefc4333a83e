"""cached_block.py with experts in place of its last linears, adapters beside them, and drafted tokens that are
verified and taken back: each against a 64-bit recomputation."""
import numpy as np
import pytest
import torch

import b2q
import cached_block as cb
import oracle as O
from test_gpu_cached_block import coords, layer_norm, reference

pytestmark = pytest.mark.gpu

C, HEADS, D, HIDDEN = 256, 4, 64, 512
SECTIONS = (12, 10, 10)


def values(raw, n, k, dev):
    return torch.from_numpy(O.dequantize(raw, O.TYPE_Q4_0, k)).double().to(dev).view(n, k)


def experts_reference(h, raws, E, F, top):
    """The mixture layer of normed rows h (fp64)."""
    router, w_in, w_out = raws
    dev = h.device
    w1 = values(w_in, E * 2 * F, C, dev).view(E, 2 * F, C)
    w2 = values(w_out, E * C, F, dev).view(E, C, F)
    logits = h @ torch.from_numpy(router).double().to(dev).t()
    best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    share = torch.softmax(best[:, :top], 1)
    out = torch.zeros_like(h)
    for t in range(h.shape[0]):
        for j in range(top):
            z = w1[ids[t, j]] @ h[t]
            out[t] += share[t, j] * (w2[ids[t, j]] @ (z[:F] * torch.sigmoid(z[:F]) * z[F:]))
    return out, (best[:, top - 1] - best[:, top]).min()


@pytest.mark.parametrize("tokens", [1, 7, 90])
def test_experts_layer(dev, tokens):
    """Rows in fp16 (h and the hidden values, 2^-11 each), everything else fp32 or exact."""
    E, F, top = 8, 160, 3
    experts, raws = cb.random_experts(dev, E, C, F, top, seed=tokens)
    g = torch.Generator(device=dev).manual_seed(tokens)
    x = torch.randn(tokens, C, generator=g, device=dev)
    h = layer_norm(x.double())
    ref, gap = experts_reference(h, raws, E, F, top)
    assert float(gap) > 1e-5  # the choice does not hang on the router's rounding
    y = experts.forward(b2q.norm_modulate(x), x.clone())
    err = (y.double() - x.double() - ref).norm() / ref.norm()
    assert float(err) <= 2.0 ** -9


def test_block_with_experts_steps_match_their_own_prompt(dev):
    """Tokens one by one through attention and experts give what the whole prompt at once gives."""
    experts, _ = cb.random_experts(dev, 6, C, 96, 2, seed=2)
    block, _ = cb.random_block(dev, C, HEADS, HEADS, D, HIDDEN, SECTIONS, seed=3, experts=experts, unrounded_rows=64)
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(30, C, generator=g, device=dev)
    cache = cb.PagedCache(dev, 1, 1, HEADS, D, pages=4, page_size=16, max_len=64)
    step = cache.plan([30])
    whole = block.forward(x.clone(), cache, 0, step, coords(step["pos"]))
    cache = cb.PagedCache(dev, 1, 1, HEADS, D, pages=4, page_size=16, max_len=64)
    rows = []
    for i in range(30):
        step = cache.plan([1])
        rows.append(block.forward(x[i:i + 1].clone(), cache, 0, step, coords(step["pos"])))
    err = (torch.cat(rows) - whole).norm() / (whole - x).norm()
    assert float(err) <= 4e-3  # fp16 q, k, v, o and rows, as of the block without experts


@pytest.mark.parametrize("counts", [[2, 3], [70, 41]])
def test_block_with_adapters(dev, counts):
    """Each request's adapter merged into the weights of its own 64-bit recomputation; one request has none."""
    G, rank = 3, 16
    block, weights = cb.random_block(dev, C, HEADS, HEADS, D, HIDDEN, SECTIONS, seed=5, unrounded_rows=128)
    g = torch.Generator(device=dev).manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    pairs = {n: ((r(G, rank, k) / k ** 0.5).half(), (0.3 * r(G, out, rank) / rank ** 0.5).half())
             for n, (out, k) in block.shape.items()}
    adapters = cb.Adapters(pairs, torch.tensor([0.5, 1.0, 2.0], device=dev))
    counts = counts + [3]
    mine = [2, 0, -1]
    xs = [r(n, C) for n in counts]
    ids = torch.repeat_interleave(torch.tensor(mine), torch.tensor(counts)).int().to(dev)
    cache = cb.PagedCache(dev, 1, 3, HEADS, D, pages=20, page_size=16, max_len=128)
    step = cache.plan(counts)
    y = block.forward(torch.cat(xs), cache, 0, step, coords(step["pos"]), adapters=adapters, rows=adapters.plan(ids))
    plain = block.forward(torch.cat(xs), cache, 0, step, coords(step["pos"]))
    at = 0
    for b, x in enumerate(xs):
        if mine[b] < 0:
            assert torch.equal(y[at:at + counts[b]], plain[at:at + counts[b]])
        ref = merged_reference(block, weights, x, pairs, adapters.scales, mine[b])
        got = y[at:at + counts[b]].double() - x.double()
        assert float((got - ref).norm() / ref.norm()) <= 4e-3
        at += counts[b]


def merged_reference(block, weights, x, pairs, scales, a):
    """test_gpu_cached_block's reference with W + s b a in the place of W."""
    real = O.dequantize

    def merged(raw, wtype, k):
        w = real(raw, wtype, k)
        for n, r in weights.items():
            if r is raw and a >= 0:
                low, up = pairs[n]
                w = w.astype(np.float64) + float(scales[a]) * (up[a].double() @ low[a].double()).cpu().numpy()
        return w

    O.dequantize = merged
    try:
        grid = coords(torch.arange(x.shape[0], device=x.device))
        return reference(block, weights, x.double(), grid) - x.double()
    finally:
        O.dequantize = real


def test_drafts_are_verified_and_taken_back(dev):
    """A step of drafted tokens, their verification, and the cache taken back: the next step goes on as if only the
    kept tokens had ever been added."""
    block, _ = cb.random_block(dev, C, HEADS, HEADS, D, HIDDEN, SECTIONS, seed=6, unrounded_rows=64)
    V = 50
    g = torch.Generator(device=dev).manual_seed(3)
    embed, head = torch.randn(V, C, generator=g, device=dev), torch.randn(V, C, generator=g, device=dev) / 16
    prompts = [[3, 1, 4, 1, 5], [9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2, 3, 8, 4]]

    def run(cache, tokens):
        step = cache.plan([len(t) for t in tokens])
        x = embed[torch.tensor(sum(tokens, []), device=dev)].clone()
        return torch.softmax(block.forward(x, cache, 0, step, coords(step["pos"])) @ head.t(), -1)

    cache = cb.PagedCache(dev, 1, 2, HEADS, D, pages=6, page_size=16, max_len=64)
    run(cache, [p[:-1] for p in prompts])
    drafts = [[7, 7, 7, 7, 7], [1, 2, 3]]
    probs = run(cache, [[p[-1]] + d for p, d in zip(prompts, drafts)])  # the last token and the drafts behind it
    cu = torch.tensor([0, 5, 8], dtype=torch.int32, device=dev)
    flat = torch.tensor(sum(drafts, []), dtype=torch.int32, device=dev)
    u = torch.tensor([0.0, 0.0, 0.999, 0.0, 0.0, 0.0, 0.0, 0.0], device=dev)  # the third of the first request goes
    accepted, tokens = b2q.draft_verify(probs, None, flat, cu, u, torch.full((2,), 0.5, device=dev))
    assert accepted.tolist() == [2, 3]
    kept = [p + d[:n] for p, d, n in zip(prompts, drafts, accepted.tolist())]
    taken = cache.taken
    for b in range(2):
        cache.keep(b, len(kept[b]))
    assert cache.lengths == [len(k) for k in kept] and cache.taken == taken  # (request 1 fills 18 of 32 places)
    new = [int(tokens[2]), int(tokens[9])]
    assert all(0 <= n < V for n in new) and new[0] != 7 and tokens[3:6].tolist() == [-1] * 3
    after = run(cache, [[n] for n in new])
    fresh = cb.PagedCache(dev, 1, 2, HEADS, D, pages=6, page_size=16, max_len=64)
    want = run(fresh, [k + [n] for k, n in zip(kept, new)])
    ends = np.cumsum([len(k) + 1 for k in kept]) - 1
    # the same arithmetic over the same keys, in another order of sums: fp16 q, k, v and o
    assert float((after - want[torch.from_numpy(ends).to(dev)]).abs().max()) <= 2e-3


def test_pages_behind_the_kept_tokens_are_free_again(dev):
    cache = cb.PagedCache(dev, 1, 2, 1, 64, pages=8, page_size=16, max_len=96)
    cache.plan([20, 60])
    assert cache.taken == 6
    cache.keep(1, 17)
    assert cache.taken == 4 and cache.lengths == [20, 17]
    assert cache.table[1].tolist()[2:] == [-1] * 4
    cache.keep(1, 17)
    cache.keep(0, 0)
    assert cache.taken == 2 and cache.table[0].tolist() == [-1] * 6
    cache.plan([96, 0])
    used = [p for p in cache.table.flatten().tolist() if p >= 0]
    assert len(used) == len(set(used)) == 8
    for bad in (-1, 97):
        with pytest.raises(ValueError):
            cache.keep(0, bad)
