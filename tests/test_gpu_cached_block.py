"""The block over a paged cache (cached_block.py): prompts and single tokens of
several requests, against a 64-bit recomputation of each whole request without
a cache."""
import math

import numpy as np
import pytest
import torch

import b2q
import cached_block as cb
import oracle as O

pytestmark = pytest.mark.gpu

EPS = 1e-6


def layer_norm(x):
    d = x - x.mean(-1, keepdim=True)
    return d / torch.sqrt(d.square().mean(-1, keepdim=True) + EPS)


def reference(block, weights, x, grid):
    """One request's tokens x [n, C] (fp64) through the block, causal, no cache."""
    dev = x.device
    w = {n: torch.from_numpy(O.dequantize(weights[n], O.TYPE_Q4_0, k)).double().to(dev) for n, (_, k) in block.shape.items()}
    v = {n: t.double() for n, t in block.vec.items()}
    n, H, Hk, D = x.shape[0], block.H, block.Hk, block.D
    qkv = layer_norm(x) @ w["qkv"].t() + v["b_qkv"]
    q, k, vv = qkv.view(n, H + 2 * Hk, D).split([H, Hk, Hk], 1)
    rms = lambda t, g: t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * g.view(-1, D)  # noqa: E731
    axis = torch.repeat_interleave(torch.arange(3, device=dev), torch.tensor(block.sections, device=dev))
    th = grid.double()[axis].t() * block.inv_freq.double()
    c, s = torch.cos(th)[:, None], torch.sin(th)[:, None]

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, k = turn(rms(q, v["gq"])), turn(rms(k, v["gk"]))
    i, j = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None]
    see = j <= i
    if block.window:
        see &= (j > i - block.window) | (j < block.sinks)
    o = []
    for h in range(H):
        sc = (q[:, h] @ k[:, h // (H // Hk)].t()) / D ** 0.5
        o.append(torch.softmax(sc.masked_fill(~see, float("-inf")), -1) @ vv[:, h // (H // Hk)])
    x = x + torch.cat(o, 1) @ w["out"].t() + v["b_out"]
    h = layer_norm(x) @ w["fc1"].t() + v["b1"]
    h = 0.5 * h * (1 + torch.tanh(0.7978845608028654 * (h + 0.044715 * h ** 3)))
    return x + h @ w["fc2"].t() + v["b2"]


def coords(p):
    return torch.stack([p // 64, p // 8 % 8, p % 8]).int()


@pytest.mark.parametrize("heads,kv_heads,D,window,sinks", [(4, 4, 64, 0, 0), (6, 2, 64, 20, 3), (4, 1, 128, 0, 0)])
@pytest.mark.parametrize("steps,bound", [
    # Steps of at most 8 tokens in all: q, k, v and o are rounded to fp16 (2^-11 each) and gelu
    # runs on fp16 inputs and outputs as ggml's does; everything else is fp32.
    ([[3, 5], [1, 1], [1, 1], [2, 6], [1, 0], [4, 4], [0, 1], [1, 1]], 4e-3),
    # Chunks too: their linears round the activations to Q8_0, half of 1/127 of a block's largest value.
    ([[70, 133], [1, 1], [1, 1], [40, 3], [1, 1]], 2e-2),
])
def test_cached_steps_match_full_recomputation(dev, heads, kv_heads, D, window, sinks, steps, bound):
    C, hidden = 256, 512
    sections = (D // 2 - 2 * (D // 8), D // 8, D // 8)
    block, weights = cb.random_block(dev, C, heads, kv_heads, D, hidden, sections, seed=3, window=window, sinks=sinks)
    total = [sum(s[b] for s in steps) for b in range(2)]
    g = torch.Generator(device=dev).manual_seed(1)
    xs = [torch.randn(n, C, generator=g, device=dev) for n in total]
    refs = [reference(block, weights, x.double(), coords(torch.arange(x.shape[0], device=dev))) for x in xs]
    cache = cb.PagedCache(dev, 1, 2, kv_heads, D, pages=40, page_size=16, max_len=320)
    at = [0, 0]
    for new in steps:
        step = cache.plan(new)
        x = torch.cat([xs[b][at[b]:at[b] + new[b]] for b in range(2)])
        y = block.forward(x.clone(), cache, 0, step, coords(step["pos"]))
        ref = torch.cat([refs[b][at[b]:at[b] + new[b]] for b in range(2)])
        err = (y.double() - ref).norm() / (ref - x.double()).norm()
        assert float(err) <= bound, (new, float(err))
        at = [at[b] + new[b] for b in range(2)]


def test_full_cache_is_refused(dev):
    cache = cb.PagedCache(dev, 1, 1, 1, 64, pages=2, page_size=16, max_len=64)
    cache.plan([30])
    with pytest.raises(RuntimeError):
        cache.plan([3])
    cache = cb.PagedCache(dev, 1, 1, 1, 64, pages=20, page_size=16, max_len=32)
    with pytest.raises(RuntimeError):
        cache.plan([33])


def test_example_runs(dev, capsys):
    cb.main()
    out = capsys.readouterr().out.splitlines()
    assert len(out) == 9 and out[-1].endswith("cached 308")
    assert all(np.isfinite(float(line.split("rms ")[1].split(",")[0])) for line in out)


def test_results_on_another_stream_come_from_its_pool(dev):
    """Outputs and workspaces of a call on a given stream are allocated for it: memory that the current stream
    has freed, and still works on, is not handed to the other one."""
    D, n = 128, 30011
    kc = torch.randn(n // 16 + 1, 1, 16, D, device=dev).half()
    vc = torch.randn_like(kc)
    table = torch.arange(kc.shape[0], dtype=torch.int32, device=dev)[None]
    kv_len = torch.tensor([n], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    q = torch.randn(1, 2 * D, device=dev).half()
    assert b2q.attention_paged_workspace_bytes(1, 1, 1, n, 2, 1, D) > 0
    ref = b2q.attention_paged(q, kc, vc, table, kv_len, cu, 1, n, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(8192, 8192, device=dev)
    for _ in range(4):
        for _ in range(4):
            big = torch.tanh(big @ big)                              # the current stream is busy,
        scrap = torch.full((1 << 20,), math.nan, device=dev)         # and then writes what it has freed by now
        del scrap
        o = b2q.attention_paged(q, kc, vc, table, kv_len, cu, 1, n, 2, stream=side)
        side.synchronize()
        assert torch.equal(o, ref)
    torch.cuda.synchronize()


@pytest.mark.parametrize("news", [[[40, 30], [2, 1], [1, 1]]])
def test_forward_on_another_stream(dev, news):
    """Steps of more than eight tokens and of few, plan and forward on a given stream, while the current stream is
    busy: the results of the same steps on the current stream."""
    C, heads, D, hidden = 256, 4, 64, 512
    block, _ = cb.random_block(dev, C, heads, heads, D, hidden, (12, 10, 10), seed=4)
    g = torch.Generator(device=dev).manual_seed(2)
    xs = [torch.randn(sum(n), C, generator=g, device=dev) for n in news]
    grids = []

    def steps(stream=None, before=lambda: None):
        cache = cb.PagedCache(dev, 1, 2, heads, D, pages=16, page_size=16, max_len=64)
        torch.cuda.synchronize()
        out = []
        for i, (n, x0) in enumerate(zip(news, xs)):
            x = x0.clone()
            torch.cuda.synchronize()
            before()
            step = cache.plan(n, stream=stream)
            if stream is None:
                grids.append(coords(step["pos"]))
            out.append(block.forward(x, cache, 0, step, grids[i], stream=stream))
            if stream is not None:
                stream.synchronize()
        torch.cuda.synchronize()
        return [y.clone() for y in out]

    ref = steps()
    side = torch.cuda.Stream()
    big = torch.randn(8192, 8192, device=dev)

    def busy():  # what the current stream's pool hands out from here on holds NaN, and the stream has work for long
        nonlocal big
        held = [torch.full((rows * cols,), math.nan, device=dev) for rows in (70, 3, 2) for cols in (C, 768, hidden) for _ in range(40)]
        torch.cuda.synchronize()
        del held
        for _ in range(8):
            big = torch.tanh(big @ big)

    for a, b in zip(steps(side, busy), ref):
        assert torch.equal(a, b)


def test_operands_on_the_host_are_refused(dev):
    """Addresses of the host's memory never reach a kernel."""
    i32 = lambda n, d=dev: torch.zeros(n, dtype=torch.int32, device=d)  # noqa: E731
    table, pool = i32((2, 4)), torch.zeros(4, 1, 16, 64, dtype=torch.float16, device=dev)
    for bad in range(3):
        lens = [i32(2, "cpu" if bad == i else dev) for i in range(3)]
        with pytest.raises(AssertionError):
            b2q.kv_cache_plan(lens[0], lens[1], 16, lens[2], table, 2)
    qkv, inv = torch.zeros(2, 3 * 64, device=dev), torch.zeros(32, device=dev)
    for bad in range(3):
        pos, f, slots = i32((1, 2)), inv, torch.zeros(2, dtype=torch.int64, device=dev)
        pos, f, slots = (t.cpu() if bad == i else t for i, t in enumerate((pos, f, slots)))
        with pytest.raises(AssertionError):
            b2q.qkv_rope_cache(qkv, 1, 1, 64, pos, (32,), f, slots, pool, pool.clone())
    q = torch.zeros(2, 64, dtype=torch.float16, device=dev)
    for bad in range(3):
        ops = [t.cpu() if bad == i else t for i, t in enumerate((table, i32(2), i32(3)))]
        with pytest.raises(AssertionError):
            b2q.attention_paged(q, pool, pool, *ops, 1, 16, 1)
    packed = b2q.weight_pack_q4_0(torch.zeros(16, 18, dtype=torch.uint8, device=dev), 32)
    with pytest.raises(AssertionError):
        b2q.mul_vec(b2q.TYPE_Q4_0, packed, 16, 32, torch.zeros(1, 32, device=dev), bias=torch.zeros(16))
    assert b2q.device_status() == 0


def test_negative_counts_are_refused(dev):
    """The device takes a negative count for none; the host's lengths must not shrink beside it."""
    cache = cb.PagedCache(dev, 1, 2, 1, 64, pages=8, page_size=16, max_len=64)
    cache.plan([20, 3])
    with pytest.raises(ValueError):
        cache.plan([-4, 1])
    assert cache.lengths == [20, 3]
    assert cache.plan([1, 0])["kv_len"].tolist() == [21, 3]


def test_plan_does_not_wait_for_the_device(dev):
    cache = cb.PagedCache(dev, 1, 2, 1, 64, pages=8, page_size=16, max_len=64)
    for _ in range(3):
        cache.plan([1, 2])  # memory of these sizes is at hand from here on
    torch.cuda.synchronize()
    big = torch.randn(8192, 8192, device=dev)
    done = torch.cuda.Event()
    for _ in range(8):
        big = torch.tanh(big @ big)
    done.record()
    step = cache.plan([2, 1])
    assert not done.query()
    assert step["kv_len"].tolist() == [5, 7] and step["pos"].tolist() == [3, 4, 6]


def test_released_pages_serve_other_requests(dev):
    """More requests than the pool could hold, one after another: every page has one owner, and steps on pages that
    others have left match a recomputation without a cache."""
    C, heads, D, hidden = 256, 4, 64, 512
    block, weights = cb.random_block(dev, C, heads, heads, D, hidden, (12, 10, 10), seed=5)
    cache = cb.PagedCache(dev, 1, 3, heads, D, pages=9, page_size=16, max_len=64)
    g = torch.Generator(device=dev).manual_seed(6)
    rng = np.random.default_rng(7)
    xs = [torch.zeros(0, C, device=dev) for _ in range(3)]
    for turn in range(12):
        new = [int(n) for n in rng.integers(0, 4, 3)]  # at most 8 tokens a step, as mul_vec takes them
        new = [min(n, 44 - cache.lengths[b]) for b, n in enumerate(new)] if sum(new) <= 8 else [1, 1, 1]
        if sum(new) == 0:
            continue
        step = cache.plan(new)
        add = [torch.randn(n, C, generator=g, device=dev) for n in new]
        xs = [torch.cat(p) for p in zip(xs, add)]
        y = block.forward(torch.cat(add), cache, 0, step, coords(step["pos"]))
        full = [reference(block, weights, x.double(), coords(torch.arange(x.shape[0], device=dev))) for x in xs]
        ref = torch.cat([f[f.shape[0] - n:] for f, n in zip(full, new)])
        assert float((y.double() - ref).norm() / (ref - torch.cat(add).double()).norm()) <= 4e-3
        owned = cache.table[cache.table >= 0].tolist()
        left = cache.free[cache.taken:].tolist()
        assert sorted(owned + left) == list(range(9))
        b = turn % 3
        if turn % 2:
            cache.release(b)
            assert cache.lengths[b] == 0 and int(cache.table[b].max()) == -1
            assert sorted(cache.table[cache.table >= 0].tolist() + cache.free[cache.taken:].tolist()) == list(range(9))
            xs[b] = xs[b][:0]
    for _ in range(5):  # a full pool, again and again
        for b in range(3):
            cache.release(b)
        cache.plan([48, 48, 48])
        with pytest.raises(RuntimeError):
            cache.plan([1, 0, 0])
        assert sorted(cache.table[cache.table >= 0].tolist()) == list(range(9))


@pytest.mark.parametrize("requests", [9, 17])
def test_larger_batches_can_keep_their_activations(dev, requests):
    """Steps of more tokens than one product takes, with the accuracy of few: the bound for steps of at most eight."""
    C, heads, D, hidden = 256, 4, 64, 512
    block, weights = cb.random_block(dev, C, heads, heads, D, hidden, (12, 10, 10), seed=8, unrounded_rows=20)
    cache = cb.PagedCache(dev, 1, requests, heads, D, pages=requests, page_size=16, max_len=16)
    xs = torch.randn(3, requests, C, generator=torch.Generator(device=dev).manual_seed(9), device=dev)
    for t in range(3):
        step = cache.plan([1] * requests)
        y = block.forward(xs[t].clone(), cache, 0, step, coords(step["pos"]))
    ref = torch.stack([reference(block, weights, xs[:, b].double(), coords(torch.arange(3, device=dev)))[-1] for b in range(requests)])
    assert float((y.double() - ref).norm() / (ref - xs[2].double()).norm()) <= 4e-3
