"""Attention over the paged cache (b2q_attention_paged) against a 64-bit softmax,
request by request: ragged lengths, grouped heads, windows and sinks, page
sizes, missing pages, empty rows, stale memory, strides."""
import math

import pytest
import torch

import b2q

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(dev, lens, news, Hq, Hkv, D, dt, ps, seed=0, spare=2, stale=None, width=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-max(n, 0) // ps) for n in lens]
    pool = sum(need) + spare
    ids = torch.randperm(pool, generator=g, device=dev).int()
    W = max(max(need), width, 1)
    table = torch.full((len(lens), W), -1, dtype=torch.int32, device=dev)
    kc = torch.randn(pool, Hkv, ps, D, generator=g, device=dev).to(dt)
    vc = torch.randn(pool, Hkv, ps, D, generator=g, device=dev).to(dt)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    if stale is not None:  # everything that is no key of any request
        used = torch.zeros(pool, ps, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            for j in range(need[b]):
                used[table[b, j].long(), :max(0, min(ps, n - j * ps))] = True
        kc.masked_fill_(~used[:, None, :, None], stale)
        vc.masked_fill_(~used[:, None, :, None], stale)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1], Hq * D, generator=g, device=dev) * 1.5).to(dt)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    return q, kc, vc, table, i32(lens), i32(cu)


def reference(q, kc, vc, table, lens, cu, Hq, scale=None, causal=True, window=0, sinks=0):
    """(o, sum_j p_j |v_j|) in 64 bits; invisible keys are left out, not multiplied by 0."""
    P, Hkv, ps, D = kc.shape
    scale = scale if scale is not None else 1 / math.sqrt(D)
    G, dev = Hq // Hkv, q.device
    o = torch.zeros(q.shape[0], Hq, D, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(o)
    for b, L in enumerate(lens.tolist()):
        t0, t1 = int(cu[b]), int(cu[b + 1])
        L = min(max(L, 0), table.shape[1] * ps)
        n = t1 - t0
        if n == 0 or L == 0:
            continue
        j = torch.arange(L, device=dev)
        pages = table[b, j // ps].long()
        have = (pages >= 0) & (pages < P)
        i = torch.arange(n, device=dev)[:, None] + (int(lens[b]) - n)
        see = have[None] & ((j <= i) if causal else torch.ones(n, L, dtype=torch.bool, device=dev))
        if window > 0:
            see = see & ((j > i - window) | (j < sinks))
        pg = pages.clamp(0, P - 1)
        for h in range(Hkv):
            k, v = kc[pg, h, j % ps].double(), vc[pg, h, j % ps].double()
            for e in range(h * G, (h + 1) * G):
                s = (q[t0:t1, e * D:(e + 1) * D].double() @ torch.nan_to_num(k, nan=0.0).t()) * scale
                s = torch.where(see, s, torch.tensor(-math.inf, dtype=torch.float64, device=dev))
                m = s.amax(1, keepdim=True)
                p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), 0.0)
                z = p.sum(1, keepdim=True)
                p = p / torch.where(z == 0, torch.ones_like(z), z)
                clean = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
                o[t0:t1, e] = p @ clean
                mag[t0:t1, e] = p @ clean.abs()
                bad = (~torch.isfinite(v)).any(1)
                for x in torch.nonzero(bad)[:, 0].tolist():  # non-finite values reach the rows that see them
                    rows = see[:, x]
                    o[t0:t1, e][rows] += p[rows, x][:, None] * (v[x] - clean[x])[None]
    return o.view(q.shape[0], -1), mag.view(q.shape[0], -1)


def check(got, ref, mag, dt):
    """Half an ulp of the output type; P held in the type once (half an ulp of it on every term); and 2^-13 of
    the terms for fp32 scores up to 2^9 in their exponent and the hardware exp2 (2^-22)."""
    u = 2.0 ** -11 if dt == torch.float16 else 2.0 ** -8
    tol = u * ref.abs() + (u + 2.0 ** -13) * mag + 2.0 ** -24
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got))
    bad = ((got.double() - ref).abs() > tol) & fin
    assert not bool(bad.any()), float(((got.double() - ref).abs() / tol)[fin].max())


def run(dev, lens, news, Hq, Hkv, D, dt, ps, seed=0, max_kv=None, max_new=None, **kw):
    opts = {k: kw.pop(k) for k in ("scale", "causal", "window", "sinks") if k in kw}
    dt = DT[dt]
    q, kc, vc, table, L, cu = make(dev, lens, news, Hq, Hkv, D, dt, ps, seed, **kw)
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news) if max_new is None else max_new,
                            max(lens) if max_kv is None else max_kv, Hq, **opts)
    ref, mag = reference(q, kc, vc, table, L, cu, Hq, **opts)
    check(o, ref, mag, dt)
    return o


# lengths of one to long ones around the unit, tile and page sizes
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_decode_lengths(dev, D, dt, ps):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4097]
    run(dev, lens, [1] * len(lens), 8, 2, D, dt, ps, seed=ps + D)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 2), (3, 1), (16, 1), (17, 1), (24, 4), (20, 4), (32, 32), (48, 2), (160, 1)])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_decode_head_groups(dev, Hq, Hkv, D, dt):
    run(dev, [700, 19, 1], [1, 1, 1], Hq, Hkv, D, dt, 32, seed=Hq)


@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "f16")])
def test_decode_split_keys(dev, D, dt):
    """Few rows over long keys: stretches of the keys on several CTAs, joined afterwards; short requests beside them."""
    assert b2q.attention_paged_workspace_bytes(3, 3, 1, 30011, 4, 2, D) > 0
    run(dev, [30011, 5, 2049], [1, 1, 1], 4, 2, D, dt, 128, seed=3)


def test_announced_lengths_may_be_exceeded(dev):
    """max_kv sizes the split only: longer requests are still attended whole."""
    run(dev, [9000, 300], [1, 1], 8, 2, 64, "f16", 64, max_kv=1000)
    run(dev, [9000, 300], [1, 1], 8, 2, 64, "f16", 64, max_kv=0)
    run(dev, [900, 300], [1, 40], 8, 2, 64, "f16", 64, max_kv=100000, max_new=500)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("news,lens", [
    ([2, 3, 5], [2, 40, 700]), ([7, 1, 16, 33], [7, 100, 1600, 33]), ([64, 65], [64, 1000]),
    ([127, 128, 129], [127, 500, 2000]), ([300, 1, 257], [900, 4000, 257]), ([1000], [1000]), ([513], [3001]),
])
def test_chunks(dev, D, dt, news, lens):
    run(dev, lens, news, 8, 2, D, dt, 64, seed=len(news))


@pytest.mark.parametrize("ps", [16, 32, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 1, 64), (6, 6, 128), (10, 2, 128), (7, 1, 128), (16, 16, 64)])
def test_chunk_pages_and_groups(dev, ps, Hq, Hkv, D):
    run(dev, [333, 1471, 200], [333, 150, 199], Hq, Hkv, D, "f16", ps, seed=ps + Hq)


@pytest.mark.parametrize("news,lens", [([1, 1, 1], [5000, 100, 17]), ([3, 6], [3000, 40]), ([200, 333], [200, 2500])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 37), (1000, 130), (6000, 4), (64, 5000)])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_window_and_sinks(dev, news, lens, window, sinks, D, dt):
    run(dev, lens, news, 6, 2, D, dt, 32, seed=window, window=window, sinks=sinks)


@pytest.mark.parametrize("news,lens", [([1, 1], [900, 3]), ([5, 17], [64, 900]), ([300, 129], [1374, 129])])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_not_causal(dev, news, lens, D, dt):
    run(dev, lens, news, 4, 2, D, dt, 64, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 4.0])
def test_scales(dev, scale):
    """Weights from uniform to those of a single key; a negative scale turns the order around."""
    run(dev, [300, 900, 64], [1, 4, 40], 4, 2, 64, "f16", 16, scale=scale)
    run(dev, [300, 900], [200, 130], 4, 2, 128, "bf16", 64, scale=scale)


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [3, 2, 20, 6], [150, 130, 40, 300]])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_nothing(dev, news, D):
    """No keys, fewer keys than new tokens (negative positions), no new tokens, absent pages: zeros, and no NaN."""
    lens = [0, max(1, news[1] // 2), 500, 700]
    dt = torch.float16
    q, kc, vc, table, L, cu = make(dev, lens, news, 4, 2, D, dt, 32, stale=float("nan"))
    table[2] = -1
    table[3, 2:5] = -1
    table[3, 7] = kc.shape[0] + 5  # outside the pool: absent too
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 4)
    ref, mag = reference(q, kc, vc, table, L, cu, 4)
    check(o, ref, mag, dt)
    assert bool((o[:news[0]] == 0).all()) and bool((o[int(cu[2]):int(cu[3])] == 0).all())


@pytest.mark.parametrize("news,lens", [([1, 1, 1], [37, 129, 700]), ([5, 3, 9], [37, 129, 700]), ([90, 140, 300], [90, 333, 700])])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("stale", [float("nan"), float("inf"), float("-inf")])
def test_stale_memory_does_not_matter(dev, news, lens, D, dt, stale):
    """NaN and infinities in every place of the pool that holds no key."""
    run(dev, lens, news, 6, 2, D, dt, 64, stale=stale)
    run(dev, lens, news, 6, 2, D, dt, 16, stale=stale, window=50, sinks=3)


@pytest.mark.parametrize("news,lens", [([6, 4], [300, 64]), ([200, 131], [500, 131])])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16"), (128, "f16")])
@pytest.mark.parametrize("v", [float("nan"), float("inf"), float("-inf")])
def test_nonfinite_keys_reach_only_rows_that_see_them(dev, news, lens, D, dt, v):
    """A later token's value, and a key that has left the window, hold an infinity or a NaN."""
    for window, sinks in ((0, 0), (40, 2)):
        dtt = DT[dt]
        q, kc, vc, table, L, cu = make(dev, lens, news, 4, 2, D, dtt, 32)
        for b in range(2):
            for key in (lens[b] - 2, lens[b] - news[b] // 2 - 1, 20):
                pg = int(table[b, key // 32])
                vc[pg, :, key % 32, 5] = v
                kc[pg, :, key % 32, 7] = float("nan") if key == lens[b] - 2 else kc[pg, :, key % 32, 7]
        o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 4, window=window, sinks=sinks)
        ref, mag = reference(q, kc, vc, table, L, cu, 4, window=window, sinks=sinks)
        # the rows that see the NaN key are NaN throughout
        for b in range(2):
            ref[int(cu[b + 1]) - 2:int(cu[b + 1])] = math.nan
        hit = ~torch.isfinite(ref)
        assert bool((~torch.isfinite(o[hit])).all())
        clean = torch.where(hit, torch.zeros_like(ref), ref)
        check(torch.where(hit, torch.zeros_like(o), o), clean, mag, dtt)


@pytest.mark.parametrize("news,lens", [([1, 1], [400, 77]), ([70, 150], [400, 150])])
def test_strides_streams_and_untouched_rows(dev, news, lens):
    Hq, Hkv, D, dt = 4, 2, 64, torch.float16
    q, kc, vc, table, L, cu = make(dev, lens, news, Hq, Hkv, D, dt, 16)
    T = q.shape[0]
    qs = torch.zeros(T + 5, Hq * D + 24, dtype=dt, device=dev)
    qs[:T, 8:8 + Hq * D] = q
    wide = torch.full((table.shape[0], table.shape[1] + 6), 10 ** 6, dtype=torch.int32, device=dev)
    wide[:, 1:1 + table.shape[1]] = table
    out = torch.full((T + 5, Hq * D + 16), 3.0, dtype=dt, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b2q.attention_paged(qs[:, 8:8 + Hq * D], kc, vc, wide[:, 1:1 + table.shape[1]], L, cu, max(news), max(lens), Hq,
                        out=out[:, :Hq * D], stream=s)
    s.synchronize()
    ref, mag = reference(q, kc, vc, table, L, cu, Hq)
    check(out[:T, :Hq * D], ref, mag, dt)
    assert bool((out[T:] == 3.0).all()) and bool((out[:, Hq * D:] == 3.0).all())  # rows past cu[B], columns past the heads


def test_bits_do_not_depend_on_the_run(dev):
    for news, lens in (([1] * 4, [20000, 3, 777, 5000]), ([100, 300], [3000, 300])):
        q, kc, vc, table, L, cu = make(dev, lens, news, 8, 2, 128, torch.bfloat16, 64)
        a = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 8)
        for _ in range(3):
            assert torch.equal(b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 8), a)


@pytest.mark.parametrize("news,lens", [([1, 1], [600, 90]), ([140, 3], [600, 90])])
def test_offsets_past_32_bits(dev, news, lens):
    """Pages whose elements lie past 2^31 in the pool."""
    Hkv, ps, D, dt = 8, 256, 128, torch.float16
    n_pages = 2 ** 31 // (Hkv * ps * D) + 8
    q, k0, v0, t0, L, cu = make(dev, lens, news, 16, Hkv, D, dt, ps, spare=0)
    kc = torch.zeros(n_pages, Hkv, ps, D, dtype=dt, device=dev)
    vc = torch.zeros_like(kc)
    shift = n_pages - k0.shape[0]
    kc[shift:], vc[shift:] = k0, v0
    table = torch.where(t0 >= 0, t0 + shift, t0)
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 16)
    ref, mag = reference(q, k0, v0, t0, L, cu, 16)
    check(o, ref, mag, dt)


def test_capture_and_new_lengths(dev):
    """One captured call serves later steps: lengths and tables are read on the device."""
    Hq, Hkv, D, dt, ps = 8, 2, 128, torch.float16, 32
    q, kc, vc, table, L, cu = make(dev, [4000, 3000], [1, 1], Hq, Hkv, D, dt, ps)
    ws = b2q._empty_aligned(max(b2q.attention_paged_workspace_bytes(2, 2, 1, 4000, Hq, Hkv, D), 256), dev)
    out = torch.zeros_like(q)
    call = lambda: b2q.attention_paged(q, kc, vc, table, L, cu, 1, 4000, Hq, out=out, ws=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lens in ([4000, 3000], [17, 2999], [1, 1]):
        L.copy_(torch.tensor(lens, dtype=torch.int32, device=dev))
        g.replay()
        ref, mag = reference(q, kc, vc, table, L, cu, Hq)
        check(out, ref, mag, dt)


# Lengths at which a call has two to eight stretches that join in one launch, one more or less, and requests that
# fill none, one or part of them; 16 rows of a kv head and 17 to 32; a share of rows that does not divide evenly.
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("Hq,Hkv,news", [(2, 2, [1, 1, 1, 0]), (16, 1, [1, 1, 1, 1]), (21, 3, [3, 1, 4, 0]), (64, 2, [1, 1, 1, 1])])
@pytest.mark.parametrize("top", [207, 208, 256, 300, 471, 512, 1100, 2047, 5100])
def test_few_stretches(dev, D, dt, Hq, Hkv, news, top):
    assert b2q.attention_paged_workspace_bytes(4, sum(news), max(news), 1100, Hq, Hkv, D) == 0
    run(dev, [top, 4, top // 2 + 1, 0 if news[3] == 0 else 1], news, Hq, Hkv, D, dt, 16, seed=top, stale=float("nan"))
    run(dev, [top, 40, 1, 7], news, Hq, Hkv, D, dt, 32, seed=top + 1, causal=False)


@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("window,sinks", [(300, 0), (700, 4), (700, 40)])
def test_few_stretches_window(dev, D, dt, window, sinks):
    run(dev, [3000, 650, 20], [5, 1, 3], 12, 2, D, dt, 64, seed=window, window=window, sinks=sinks, stale=float("inf"))


@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_few_stretches_without_pages(dev, D, dt):
    """Pages of whole stretches are missing; a request whose pages are all missing gives rows of 0."""
    q, kc, vc, table, L, cu = make(dev, [1500, 900, 600], [2, 1, 1], 8, 2, D, DT[dt], 16, seed=5)
    table[0, 10:60] = -1
    table[1, :] = -1
    table[2, 30:] = 1 << 30
    o = b2q.attention_paged(q, kc, vc, table, L, cu, 2, 1500, 8)
    ref, mag = reference(q, kc, vc, table, L, cu, 8)
    assert not bool(o[2].any())
    check(o, ref, mag, DT[dt])


def test_few_stretches_nonfinite_keys(dev):
    """An infinity among the values reaches the rows that see it and no other; NaN scores give NaN rows."""
    q, kc, vc, table, L, cu = make(dev, [1200, 800], [3, 1], 8, 2, 64, torch.float16, 32, seed=6)
    vc[table[0, 1199 // 32].long(), :, 1199 % 32, 3] = math.inf   # seen by the last token only
    vc[table[1, 5].long(), 0, 2, 7] = -math.inf
    o = b2q.attention_paged(q, kc, vc, table, L, cu, 3, 1200, 8)
    ref, mag = reference(q, kc, vc, table, L, cu, 8)
    check(o, ref, mag, torch.float16)
    q[3] = math.nan
    o = b2q.attention_paged(q, kc, vc, table, L, cu, 3, 1200, 8)
    assert bool(torch.isnan(o[3]).all()) and bool(torch.isfinite(o[:2]).all())


# 33 to 128 rows of a kv head: few keys announced, and the same requests announced as long ones.
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("Hq,Hkv,news,lens", [
    (2, 2, [33, 1, 64, 0], [33, 700, 1000, 5]), (8, 1, [5, 16, 9, 12], [900, 16, 2000, 333]), (20, 2, [12, 1, 4, 7], [2036, 3, 40, 7]),
    (100, 1, [1, 1, 1, 1], [800, 1, 64, 65]),
])
@pytest.mark.parametrize("max_kv", [None, 2500])
def test_middle_numbers_of_rows(dev, D, dt, Hq, Hkv, news, lens, max_kv):
    run(dev, lens, news, Hq, Hkv, D, dt, 16, seed=Hq, max_kv=max_kv, stale=float("nan"))
    run(dev, lens, news, Hq, Hkv, D, dt, 64, seed=Hq + 1, max_kv=max_kv, window=70, sinks=3, stale=float("inf"))
    run(dev, lens, news, Hq, Hkv, D, dt, 32, seed=Hq + 2, max_kv=max_kv, causal=False)
