"""Page plan (b2q_kv_cache_plan) and qkv rows -> rotary heads + cache append
(b2q_qkv_rope_cache) against plain request-by-request / 64-bit references."""
import numpy as np
import pytest
import torch

import b2q

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------- plan
def plan_ref(cached, new, ps, free, table, max_tokens):
    """Request after request, token after token, from the definition."""
    table = table.copy()
    W = table.shape[1]
    left = max_tokens
    cu, kv, slots, pos, taken, lost = [0], [], [], [], 0, 0
    for b in range(len(cached)):
        c, n = max(int(cached[b]), 0), max(int(new[b]), 0)
        n = min(n, left)
        left -= n
        had = min(-(-c // ps), W)
        need = max(had, min(-(-(c + n) // ps), W))
        table[b, had:] = -1
        for j in range(had, need):
            if taken < len(free):
                table[b, j] = free[taken]
            taken += 1
        for p in range(c, c + n):
            page = table[b, p // ps] if p // ps < W else -1
            slots.append(int(page) * ps + p % ps if page >= 0 else -1)
            lost += page < 0
            pos.append(p)
        cu.append(cu[-1] + n)
        kv.append(c + n)
    pad = max_tokens - len(slots)
    return (table, np.array(slots + [-1] * pad, np.int64), np.array(pos + [-1] * pad, np.int32),
            np.array(cu, np.int32), np.array(kv, np.int32), np.array([taken, lost], np.int32))


def run_plan(dev, cached, new, ps, free, table, max_tokens):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)  # noqa: E731
    tab = t(table)
    out = b2q.kv_cache_plan(t(cached), t(new), ps, t(free), tab, max_tokens)
    return (tab.cpu().numpy(),) + tuple(x.cpu().numpy() for x in out)


def owned_table(rng, cached, ps, W, pool):
    ids = rng.permutation(pool).astype(np.int32)
    table = np.full((len(cached), W), -7, np.int32)  # what an unplanned column holds does not matter
    at = 0
    for b, c in enumerate(cached):
        had = min(-(-max(int(c), 0) // ps), W)
        table[b, :had] = ids[at:at + had]
        at += had
    return table, ids[at:]


@pytest.mark.parametrize("B,ps,cmax,nmax", [(1, 16, 0, 1), (1, 256, 300, 1), (3, 16, 40, 5), (64, 32, 2000, 1),
                                            (513, 16, 200, 40), (1030, 64, 900, 77), (5, 128, 1000, 3000)])
def test_plan_matches_reference(dev, B, ps, cmax, nmax):
    rng = np.random.default_rng(B * 1000 + ps)
    cached = rng.integers(0, cmax + 1, B)
    new = rng.integers(0, nmax + 1, B)
    W = (cmax + nmax) // ps + 2
    pool = int(sum(-(-(c + n) // ps) for c, n in zip(cached, new))) + 2
    table, free = owned_table(rng, cached, ps, W, pool)
    T = int(new.sum())
    got = run_plan(dev, cached, new, ps, free, table, T)
    for g, r in zip(got, plan_ref(cached, new, ps, free, table, T)):
        assert np.array_equal(g, r)


@pytest.mark.parametrize("case", ["no_free", "some_free", "narrow", "few_tokens", "spare_tokens", "negative", "no_page",
                                  "no_requests", "no_columns"])
def test_plan_shortages(dev, case):
    rng = np.random.default_rng(11)
    B, ps, W = 37, 16, 12
    cached = rng.integers(0, 100, B)
    new = rng.integers(0, 60, B)
    T = int(new.sum())
    if case == "narrow":
        W = 5
    if case == "no_columns":
        W = 0
    if case == "negative":
        cached[3], new[5], new[0] = -4, -9, -1
        T = int(np.maximum(new, 0).sum())
    if case == "no_requests":
        cached, new, T = cached[:0], new[:0], 9
    table, free = owned_table(rng, cached, ps, W, 37 * 12)
    if case == "no_free":
        free = free[:0]
    if case == "some_free":
        free = free[:20]
    if case == "few_tokens":
        T = T // 2
    if case == "spare_tokens":
        T += 101
    if case == "no_page":  # an owned page that the table lacks
        table[4, max(-(-int(cached[4]) // ps) - 1, 0)] = -1
        cached[4], new[4] = 19, 30
        T = int(new.sum())
    got = run_plan(dev, cached, new, ps, free, table, T)
    for g, r in zip(got, plan_ref(cached, new, ps, free, table, T)):
        assert np.array_equal(g, r)


def test_plan_repeats_and_strided_table(dev):
    rng = np.random.default_rng(5)
    cached, new = rng.integers(0, 400, 20), rng.integers(1, 90, 20)
    table, free = owned_table(rng, cached, 32, 16, 500)
    T = int(new.sum())
    ref = plan_ref(cached, new, 32, free, table, T)
    big = torch.full((20, 23), 123, dtype=torch.int32, device=dev)
    view = big[:, 2:18]
    view.copy_(torch.from_numpy(table))
    t = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(dev)  # noqa: E731
    for _ in range(2):  # a repeated call gives the same plan
        out = b2q.kv_cache_plan(t(cached), t(new), 32, t(free), view, T)
        assert np.array_equal(view.cpu().numpy(), ref[0])
        for g, r in zip(out, ref[1:]):
            assert np.array_equal(g.cpu().numpy(), r)
    assert bool((big[:, :2] == 123).all()) and bool((big[:, 18:] == 123).all())


def test_plan_most_requests(dev):
    B = 16384
    rng = np.random.default_rng(8)
    cached, new = rng.integers(0, 40, B), rng.integers(0, 4, B)
    table, free = owned_table(rng, cached, 16, 3, 3 * B)
    T = int(new.sum())
    got = run_plan(dev, cached, new, 16, free, table, T)
    for g, r in zip(got, plan_ref(cached, new, 16, free, table, T)):
        assert np.array_equal(g, r)


# ------------------------------------------------------------------------------------------------------------- rope
def rope_ref(qkv, Hq, Hkv, D, pos, sections, inv_freq, norm, gq, gk, eps, inter):
    """q, k, v in 64 bits, and the sum of magnitudes that each rotated value is made of."""
    T = qkv.shape[0]
    x = qkv.double().view(T, Hq + 2 * Hkv, D)
    h = x[:, :Hq + Hkv]
    if norm:
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
        g = torch.ones(Hq + Hkv, D, dtype=torch.float64, device=qkv.device)
        if gq is not None:
            g[:Hq] = gq.double().view(Hq, D)
        if gk is not None:
            g[Hq:] = gk.double().view(Hkv, D)
        h = h * g
    out, mag = h.clone(), h.abs()
    R, i = sum(sections), 0
    for axis, n in enumerate(sections):
        for _ in range(n):
            a, b = (2 * i, 2 * i + 1) if inter else (i, i + R)
            th = pos[axis].double() * inv_freq[i].double()
            c, s = torch.cos(th)[:, None], torch.sin(th)[:, None]
            out[:, :, a] = h[:, :, a] * c - h[:, :, b] * s
            out[:, :, b] = h[:, :, b] * c + h[:, :, a] * s
            m = h[:, :, a].abs() + h[:, :, b].abs()
            mag[:, :, a] = m
            mag[:, :, b] = m
            i += 1
    return out[:, :Hq].reshape(T, -1), out[:, Hq:], x[:, Hq + Hkv:], mag


def close16(got, ref, mag, dt):
    """One rounding to the type (half an ulp, 2^-11 or 2^-8 relative; 2^-25 absolute for fp16's
    subnormals) of a value that fp32 arithmetic leaves within 16 roundings (2^-20) of its terms."""
    u = 2.0 ** -11 if dt == torch.float16 else 2.0 ** -8
    tol = u * ref.abs() + 2.0 ** -20 * mag + 2.0 ** -25
    assert bool(((got.double() - ref).abs() <= tol * (1 + 1e-6)).all())


@pytest.mark.parametrize("T,Hq,Hkv,D,sections,inter,norm,dt,ps", [
    (1, 1, 1, 64, (32,), False, False, "f16", 16),
    (1, 24, 8, 128, (22, 21, 21), False, True, "bf16", 64),
    (3, 5, 1, 64, (16, 8, 8), True, False, "bf16", 32),
    (37, 16, 16, 64, (12, 10, 10), True, True, "f16", 256),
    (130, 8, 2, 128, (64,), False, True, "f16", 128),
    (1201, 6, 3, 128, (32, 32), True, False, "bf16", 16),
    (2500, 4, 4, 64, (10, 10, 8), False, True, "f16", 16),   # 28 of 32 pairs, partners four lanes' width apart
    (700, 3, 1, 64, (3, 2, 2), False, True, "f16", 32),      # 7 pairs: partners across lanes
    (11, 2, 1, 128, (7, 0, 6), True, True, "bf16", 32),      # an axis without pairs
    (9, 2, 2, 64, (), False, True, "f16", 16),               # no rotation
    (19, 4, 0, 64, (32,), False, False, "f16", 16),          # q only
    (19, 0, 3, 128, (64,), False, False, "f16", 16),         # k and v only
])
def test_rope_cache(dev, T, Hq, Hkv, D, sections, inter, norm, dt, ps):
    g = torch.Generator(device=dev).manual_seed(T * 7 + Hq)
    dt = torch.float16 if dt == "f16" else torch.bfloat16
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device=dev) * 2
    R = sum(sections)
    pos = torch.randint(-50, 20000, (len(sections), T), generator=g, device=dev, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(R, device=dev, dtype=torch.float32) / max(R, 1))
    gq = 1 + 0.3 * torch.randn(Hq * D, generator=g, device=dev) if norm and T % 2 else None
    gk = 1 + 0.3 * torch.randn(Hkv * D, generator=g, device=dev) if norm else None
    n_pages = -(-T // ps) + 3
    slots = torch.randperm(n_pages * ps, generator=g, device=dev)[:T].contiguous()
    if T > 8:
        slots[3], slots[7] = -1, n_pages * ps  # neither is written
    kc = torch.full((n_pages, Hkv, ps, D), 7.0, dtype=dt, device=dev)
    vc = torch.full((n_pages, Hkv, ps, D), -7.0, dtype=dt, device=dev)
    q = b2q.qkv_rope_cache(qkv, Hq, Hkv, D, pos, sections, inv, slots, kc, vc, norm=norm, gamma_q=gq, gamma_k=gk,
                           eps=1e-5, interleaved=inter)
    rq, rk, rv, mag = rope_ref(qkv, Hq, Hkv, D, pos, sections, inv, norm, gq, gk, 1e-5, inter)
    close16(q, rq, mag[:, :Hq].reshape(T, -1), dt)
    flat = lambda c: c.transpose(1, 2).reshape(n_pages * ps, Hkv, D)  # noqa: E731
    ok = (slots >= 0) & (slots < n_pages * ps)
    close16(flat(kc)[slots[ok]], rk[ok], mag[ok][:, Hq:], dt)
    assert torch.equal(flat(vc)[slots[ok]], rv[ok].float().to(dt))
    rest = torch.ones(n_pages * ps, dtype=torch.bool, device=dev)
    rest[slots[ok]] = False
    assert bool((flat(kc)[rest] == 7.0).all()) and bool((flat(vc)[rest] == -7.0).all())


def test_rope_strides_and_stream(dev):
    T, Hq, Hkv, D = 65, 3, 1, 64
    wide = torch.randn(T, 5 * D + 12, device=dev)
    out = torch.zeros(T, Hq * D + 8, dtype=torch.float16, device=dev)
    pos = torch.arange(T, device=dev, dtype=torch.int32)[None]
    inv = 10000.0 ** (-torch.arange(32, device=dev, dtype=torch.float32) / 32)
    kc, vc = (torch.zeros(5, Hkv, 16, D, dtype=torch.float16, device=dev) for _ in range(2))
    slots = torch.arange(T, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b2q.qkv_rope_cache(wide[:, 4:4 + 5 * D], Hq, Hkv, D, pos, (32,), inv, slots, kc, vc, out=out[:, :Hq * D], stream=s)
    s.synchronize()
    rq, rk, _, mag = rope_ref(wide[:, 4:4 + 5 * D].contiguous(), Hq, Hkv, D, pos, (32,), inv, False, None, None, 0, False)
    close16(out[:, :Hq * D], rq, mag[:, :Hq].reshape(T, -1), torch.float16)
    assert bool((out[:, Hq * D:] == 0).all())


def test_rope_far_positions(dev):
    """Positions near 2^31: the angle is reduced before it is rounded."""
    T, D = 64, 64
    qkv = torch.randn(T, 3 * D, device=dev)
    pos = (2 ** 31 - 1 - 977 * torch.arange(T, device=dev)).int()[None]
    inv = 10000.0 ** (-torch.arange(32, device=dev, dtype=torch.float32) / 32)
    kc, vc = (torch.zeros(4, 1, 16, D, dtype=torch.float16, device=dev) for _ in range(2))
    q = b2q.qkv_rope_cache(qkv, 1, 1, D, pos, (32,), inv, torch.arange(T, device=dev), kc, vc)
    rq, _, _, mag = rope_ref(qkv, 1, 1, D, pos, (32,), inv, False, None, None, 0, False)
    # 2^31 turns in a double carry 2^31 / 2 pi * 2^-52 of a turn: far below 2^-20 radians
    close16(q, rq, mag[:, :1].reshape(T, -1), torch.float16)


def test_rope_offsets_past_32_bits(dev):
    """Slots whose cache elements lie past 2^31."""
    Hkv, ps, D = 8, 256, 128
    n_pages = 2 ** 31 // (Hkv * ps * D) + 3
    kc = torch.zeros(n_pages, Hkv, ps, D, dtype=torch.float16, device=dev)
    vc = torch.zeros_like(kc)
    T = 5
    slots = n_pages * ps - 1 - 40 * torch.arange(T, device=dev)
    qkv = torch.randn(T, 2 * Hkv * D, device=dev)
    b2q.qkv_rope_cache(qkv, 0, Hkv, D, None, (), None, slots, kc, vc)
    x = qkv.view(T, 2 * Hkv, D).half()
    page, off = slots // ps, slots % ps
    assert torch.equal(kc[page, :, off], x[:, :Hkv]) and torch.equal(vc[page, :, off], x[:, Hkv:])
    assert int((kc[:4] != 0).sum()) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R", [2, 4, 6, 8, 12, 20, 24, 28, 30, 32])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_cache_numbers_of_pairs(dev, D, R, norm):
    """Halves of every kind of length: multiples of 4 and 8, others, and values past the pairs."""
    test_rope_cache(dev, 70, 3, 2, D, (R // 2, R - R // 2), False, norm, "bf16" if R % 8 else "f16", 16)
