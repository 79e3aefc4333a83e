"""Calls for rows that go by group at the borders between their kernels' forms, against plain 64-bit arithmetic
(tolerances as in test_gpu_groups.py, and equality where every value is exact)."""
import math
import threading

import numpy as np
import pytest
import torch

import b2q
import cached_block as cb
from test_gpu_expert_block import experts_reference as layer_reference
from test_gpu_cached_block import layer_norm
from test_gpu_groups import (DT, call_experts, call_lora, check_route, check_rows, experts_reference, lora_reference, make_experts,
                             make_lora, plan_reference)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error(dev):
    yield
    assert b2q.device_status() == 0


def slots_of(counts, dev):
    """ids [slots, 1] with that many slots of every expert, mixed up."""
    ids = torch.cat([torch.full((n,), e, dtype=torch.int32) for e, n in enumerate(counts)])
    return ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(len(counts)))].view(-1, 1).to(dev)


# K up to 1024, to 1280, to 2304 and further leave shared memory for 32, 24, 16 and 8 rows of x
@pytest.mark.parametrize("k", [1024, 1056, 1152, 1280, 1312, 2304, 2336])
@pytest.mark.parametrize("counts", [[17, 1, 0, 24], [16, 25, 8, 9], [33, 2, 7, 18], [0, 64, 0, 0]])
def test_mul_mat_id_q4_groups_of_every_number_of_tiles(dev, k, counts):
    for glu in (False, True):
        c = make_experts(dev, sum(counts), 4, 1, 40, k, "q4_0", glu, seed=k, ids=slots_of(counts, dev))
        ref, tol = experts_reference(c)
        for out in (None, torch.float32):
            check_rows(call_experts(c, out_dtype=out), ref, tol)


# --------------------------------------------------------------------------------- a bias on the router's scores
def scores_of(x, scoring):
    """fp64 scores of numpy logits; NaN and -infinity have none (-infinity)."""
    z = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if scoring == "sigmoid":
        s = 1 / (1 + np.exp(-z))
    else:
        m = np.maximum(z.max(1, keepdims=True), -1e300)
        s = np.exp(z - m)
        s /= np.maximum(s.sum(1, keepdims=True), 1e-300)
    return np.where(z == -np.inf, -np.inf, s), s


def check_scored(got, x, bias, top, scoring, renorm, scale):
    """Each choice's score + bias against the 64-bit ones: no better one left out or behind a worse one, but for the
    rounding of a score (exp of a number of at most 100, a division, a sum of E terms) and of the sum with the bias."""
    ids, weights, order, offsets = (t.cpu().numpy() for t in got)
    T, E = x.shape
    open_, score = scores_of(x, scoring)
    with np.errstate(invalid="ignore"):
        key = open_ + bias.astype(np.float64)
    key = np.where(np.isnan(key) | (open_ == -np.inf), -np.inf, key)
    tol = (E + 120) * 2.0 ** -24
    want = np.minimum((key > -np.inf).sum(1), top)
    assert np.array_equal((ids >= 0).sum(1), want) and np.all(ids[np.arange(top) >= want[:, None]] == -1)
    there = ids >= 0
    mine = np.take_along_axis(key, np.maximum(ids, 0), 1)
    best = -np.sort(-key, axis=1)[:, :top]
    slack = 2 * tol * (1 + np.abs(np.where(there, best, 0)))  # of two keys, whose scores are at most 1
    assert np.all(np.abs(np.where(there, mine, 0) - np.where(there, best, 0)) <= slack)
    assert all(len(set(r[r >= 0])) == (r >= 0).sum() for r in ids)
    w = np.where(there, np.take_along_axis(score, np.maximum(ids, 0), 1), 0.0)
    if renorm:
        w = w / np.where(w.sum(1, keepdims=True) > 0, w.sum(1, keepdims=True), 1)
    assert np.all(np.abs(weights - w * scale) <= 2 * tol * np.abs(w * scale) + 1e-37)
    ro, rf = plan_reference(ids, E)
    assert np.array_equal(order, ro) and np.array_equal(offsets, rf)


@pytest.mark.parametrize("T,E,top", [(1, 1, 1), (12, 64, 6), (33, 33, 4), (700, 160, 8), (4097, 31, 3), (513, 1024, 32), (90, 200, 8),
                                     (9, 300, 32)])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_route_bias_on_scores(dev, T, E, top, ty):
    g = torch.Generator(device=dev).manual_seed(T + E)
    x = (2 * torch.randn(T, E, generator=g, device=dev)).to(DT[ty])
    bias = 0.3 * torch.randn(E, generator=g, device=dev)
    n = x.float().cpu().numpy()
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = b2q.moe_route(x, top, bias=bias, scoring=scoring, renorm=renorm, scale=2.5, bias_on="score")
            check_scored(got, n, bias.cpu().numpy(), top, scoring, renorm, 2.5)
            plain = b2q.moe_route(x, top, scoring=scoring, renorm=renorm, scale=2.5)
            none = b2q.moe_route(x, top, scoring=scoring, renorm=renorm, scale=2.5, bias_on="score")
            assert all(torch.equal(p, q) for p, q in zip(plain, none))


def test_route_bias_on_scores_is_another_choice(dev):
    """A bias of 0.1 puts a sigmoid score of 0.95 in front of one of 0.99, whose logit it could not reach."""
    x = torch.tensor([[math.log(99), math.log(19), 0.0]], device=dev)  # scores 0.99, 0.95, 0.5
    bias = torch.tensor([0.0, 0.1, 0.0], device=dev)
    assert b2q.moe_route(x, 1, bias=bias, scoring="sigmoid", bias_on="score")[0].tolist() == [[1]]
    assert b2q.moe_route(x, 1, bias=bias, scoring="sigmoid")[0].tolist() == [[0]]


@pytest.mark.parametrize("T", [5, 1500])
def test_route_bias_on_scores_of_masked_experts(dev, T):
    """-infinity and NaN are not chosen however large their bias; a bias of -infinity or NaN takes an expert out."""
    E, top = 40, 6
    rng = np.random.default_rng(5)
    x = rng.standard_normal((T, E)).astype(np.float32)
    x[0, ::3] = np.nan
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = -np.inf
    x[3, [7, 30]] = [1.0, 2.0]
    x[4, 5:] = -np.inf
    bias = (0.2 * rng.standard_normal(E)).astype(np.float32)
    bias[[0, 3, 6, 11]] = 5.0
    bias[9], bias[14] = -np.inf, np.nan
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = b2q.moe_route(torch.from_numpy(x).to(dev), top, bias=torch.from_numpy(bias).to(dev), scoring=scoring,
                                renorm=renorm, bias_on="score")
            check_scored(got, x, bias, top, scoring, renorm, 1.0)


def test_experts_take_a_correction_bias_on_the_scores(dev):
    experts, (router, _, _) = cb.random_experts(dev, 8, 64, 32, 2, scoring="sigmoid", bias=None)
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(50, 64, generator=g, device=dev)
    h = b2q.norm_modulate(x)
    logits = b2q.mul_mat_f32(experts.router, h)
    bias = 0.4 * torch.randn(8, generator=g, device=dev)
    ids, shares, _, _ = b2q.moe_route(logits, 2, bias=bias, scoring="sigmoid", bias_on="score")
    assert not torch.equal(ids, b2q.moe_route(logits, 2, bias=bias, scoring="sigmoid")[0])
    experts.bias = bias
    got = experts.forward(h, x.clone())
    order, offsets = b2q.group_rows(ids, 8)
    z = b2q.mul_mat_id(b2q.TYPE_Q4_0, experts.w_in, 32, 64, h.half(), order, offsets, per_row=2, glu=True)
    y = b2q.mul_mat_id(b2q.TYPE_Q4_0, experts.w_out, 64, 32, z, order, offsets, out_dtype=torch.float32)
    assert torch.equal(got, b2q.moe_combine(y, shares, ids, resid=x))


# ----------------------------------------------------------------------------- values beyond fp16's range in a block
def scaled_q4_0(raw, by):
    """GGUF Q4_0 rows times a power of two."""
    rows, width = raw.shape
    raw = raw.reshape(rows, width // 18, 18).copy()
    raw[:, :, :2] = (raw[:, :, :2].copy().view(np.float16) * np.float16(by)).view(np.uint8)
    return raw.reshape(rows, width)


@pytest.mark.parametrize("tokens", [1, 7, 90])
@pytest.mark.parametrize("big", [False, True])
def test_experts_hidden_values_beyond_fp16(dev, tokens, big):
    """Rows in fp16 of a power of two (2^-11 for h and for the hidden values), everything else fp32 or exact."""
    C, E, F, top = 256, 8, 160, 3
    experts, (router, w_in, w_out) = cb.random_experts(dev, E, C, F, top, seed=tokens)
    assert experts.hidden_fits_fp16
    if big:
        w_in = scaled_q4_0(w_in, 128.0)
        experts = cb.Experts(dev, torch.from_numpy(router).to(dev), w_in, w_out, C, F, top)
        assert not experts.hidden_fits_fp16
    g = torch.Generator(device=dev).manual_seed(tokens)
    x = torch.randn(tokens, C, generator=g, device=dev)
    h = layer_norm(x.double())
    ref, gap = layer_reference(h, (router, w_in, w_out), E, F, top)
    assert float(gap) > 1e-5
    if big:
        gates = h @ dequantized(w_in, C, dev).view(E * 2 * F, C).t()
        assert float((gates.view(tokens, E, 2, F)[:, :, 0].clamp(min=0) * gates.view(tokens, E, 2, F)[:, :, 1]).abs().max()) > 65504
    y = experts.forward(b2q.norm_modulate(x), torch.zeros_like(x))
    assert float((y.double() - ref).norm() / ref.norm()) <= 2.0 ** -9


def dequantized(raw, k, dev):
    blk = torch.from_numpy(raw).to(dev).view(raw.shape[0], k // 32, 18)
    d = blk[:, :, :2].contiguous().view(torch.float16).double()
    return (d * (torch.cat([blk[:, :, 2:] & 15, blk[:, :, 2:] >> 4], -1).double() - 8)).view(raw.shape[0], k)


def test_experts_bound_of_the_hidden_values_holds(dev):
    """A row along an expert's gate row, as long as a normed row can be."""
    C, E, F = 128, 3, 64
    _, (_, w_in, _) = cb.random_experts(dev, E, C, F, 1, seed=3)
    w = dequantized(w_in, C, dev).view(E, 2, F, C)
    bound = cb.Experts.hidden_bound(torch.from_numpy(w_in).to(dev), C, F)
    lengths = w.square().sum(-1).sqrt()
    assert abs(bound - C * float((lengths[:, 0] * lengths[:, 1]).max())) <= 1e-9 * bound
    h = w / lengths[..., None] * C ** 0.5
    gate, up = w[:, 0].flatten(0, 1), w[:, 1].flatten(0, 1)
    for rows in (h[:, 0].flatten(0, 1), h[:, 1].flatten(0, 1)):
        z = rows @ gate.t()
        assert float((z * torch.sigmoid(z) * (rows @ up.t())).abs().max()) <= bound


def test_fp16_rows(dev):
    x = torch.tensor([[1.0, -3.0, 65504.0], [1e-3, 2.0, -3.0], [0.0, 0.0, 0.0], [3e38, 1.0, -1e30], [math.inf, 1.0, 2.0],
                      [math.nan, 4.0, 5.0], [-70000.0, 3.0, 8.0]], device=dev)
    h, power = cb.fp16_rows(x)
    assert power.tolist() == [2.0, 1.0, 1.0, 2.0 ** 113, 1.0, 1.0, 4.0]
    back = h.double() * power.double()[:, None]
    fine = torch.isfinite(x)
    smallest = 2.0 ** -25 * power.double()[:, None].expand_as(x)
    assert bool(((back - x.double()).abs() <= 2.0 ** -11 * x.double().abs() + smallest)[fine].all())
    assert back[4, 0] == math.inf and bool(torch.isnan(back[5, 0]))
    assert cb.fp16_rows(x[:0])[0].shape == (0, 3)
    assert torch.equal(cb.fp16_rows(x[1:2].bfloat16())[0], x[1:2].bfloat16().half())


@pytest.mark.parametrize("dt,out", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("T,G,rank", [(5, 3, 8), (90, 4, 16), (700, 2, 64), (2500, 3, 24), (1500, 2, 128)])
def test_lora_scales_of_rows(dev, dt, out, T, G, rank):
    """Powers of two per row: what the rows give that were multiplied by them in 64 bits."""
    c = make_lora(dev, T, G, rank, 136, 77, dt, out, seed=T)
    g = torch.Generator(device=dev).manual_seed(1)
    power = 2.0 ** torch.randint(-6, 7, (T,), generator=g, device=dev).float()
    ref, tol = lora_reference(dict(c, x=c["x"].double() * power.double()[:, None]))
    y = call_lora(c, row_scales=power)
    check_rows(y, ref, tol)
    none = c["ids"] < 0
    assert torch.equal(y[none], c["resid"][none])
    assert torch.equal(call_lora(c, row_scales=torch.ones(T, device=dev)), call_lora(c))


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("name,dtype", [("fc2", torch.float32), ("out", torch.bfloat16)])
def test_adapters_rows_beyond_fp16(dev, T, name, dtype):
    """Rows in fp16 of a power of two: 2^-11 of each value, and what the smallest numbers of fp16 lose of the row's largest."""
    G, rank, k, n = 3, 16, 256, 96
    c = make_lora(dev, T, G, rank, k, n, "f16", "f32", seed=T)
    g = torch.Generator(device=dev).manual_seed(1)
    x = (torch.randn(T, k, generator=g, device=dev) * 10.0 ** (6 - torch.arange(T, device=dev)[:, None] * 3 % 10)).to(dtype)
    assert float(x.abs().max()) > 65504
    adapters = cb.Adapters({name: (c["a"], c["b"])}, c["scales"])
    y = adapters.add(name, torch.zeros(T, n, device=dev), x, adapters.plan(c["ids"]))
    exact = dict(c, x=x.double(), resid=torch.zeros(T, n, device=dev))
    ref, tol = lora_reference(exact)
    rounded = 2.0 ** -11 * x.double().abs() + 2.0 ** -25 * (x.double().abs().amax(1, keepdim=True) / 2 ** 14).clamp(min=1)
    for i in range(G):
        t = torch.nonzero(c["ids"] == i).flatten()
        tol[t] += float(c["scales"][i]) * rounded[t] @ c["a"][i].double().abs().t() @ c["b"][i].double().abs().t() * (1 + 2.0 ** -10)
    check_rows(y, ref, tol)
    small = x.abs().amax(1) < 2 ** 15  # rows that fit are taken as they were
    want = adapters.add(name, torch.zeros(T, n, device=dev), x.half(), adapters.plan(c["ids"]))
    assert torch.equal(y[small], want[small])


# ------------------------------------------------------------------------------------------- calls from two threads
@pytest.mark.parametrize("S", [400, 3000])
def test_plans_of_many_and_of_few_groups_from_two_threads(dev, S):
    """Two threads on streams of their own, one with 1024 groups, one with 400 (which need 137 KB and 53 KB of shared
    memory), in turn and at once."""
    failures = []

    def work(groups, top):
        try:
            rng = np.random.default_rng(groups)
            ids = rng.integers(-2, groups + 2, S).astype(np.int32)
            ro, rf = plan_reference(ids, groups)
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                on = torch.from_numpy(ids).to(dev)
                x = torch.from_numpy(rng.standard_normal((S // top, groups)).astype(np.float32)).to(dev)
                first = None
                for _ in range(300):
                    order, offsets = b2q.group_rows(on, groups)
                    route = b2q.moe_route(x, top)
                    first = route if first is None else first
                s.synchronize()
                assert np.array_equal(order.cpu().numpy(), ro) and np.array_equal(offsets.cpu().numpy(), rf)
                assert all(torch.equal(a, b) for a, b in zip(route, first))
        except Exception as e:  # noqa: BLE001
            failures.append((groups, repr(e)))

    for groups in (1024, 400, 1024):
        work(groups, 2)
    threads = [threading.Thread(target=work, args=(g, 2)) for g in (1024, 400, 1024, 390)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


# -------------------------------------------------------------------------------------- what is exact, to the bit
def q4_case(dev, counts, n, k, d, seed):
    """4-bit experts whose blocks have the scales d (fp16 [rows, k / 32]), x the unit rows: slot s has column 37 s."""
    E, S = len(counts), sum(counts)
    c = make_experts(dev, S, E, 1, n, k, "q4_0", seed=seed, ids=slots_of(counts, dev))
    g = torch.Generator(device=dev).manual_seed(seed)
    raw = torch.randint(0, 256, (E * n, k // 32, 18), dtype=torch.uint8, generator=g, device=dev)
    raw[:, :, :2] = d.view(torch.uint8).view(E * n, k // 32, 2)
    codes = torch.cat([raw[:, :, 2:] & 15, raw[:, :, 2:] >> 4], -1).double() - 8
    c["w64"] = (codes * d.double()[:, :, None]).view(E, n, k)
    c["w"] = b2q.weight_pack_q4_0(raw.view(E * n, -1), k)
    column = 37 * torch.arange(S, device=dev) % k
    c["x"] = torch.zeros(S, k, dtype=torch.float16, device=dev)
    c["x"][torch.arange(S, device=dev), column] = 1.0
    return c, c["w64"][c["ids"].view(-1).long(), :, column]


@pytest.mark.parametrize("counts", [[5, 9, 0, 20], [300, 41]])  # the rows kernel, and the tile kernel
@pytest.mark.parametrize("k", [64, 1408])
def test_mul_mat_id_q4_weights_are_exact(dev, counts, k):
    """Every 4-bit weight as it is: scales of 11 bits, the smallest numbers of fp16, and the largest with |8 d| < 65504."""
    n = 96
    rng = np.random.default_rng(k)
    size = (len(counts) * n, k // 32)
    ordinary = rng.uniform(0.5, 2.0, size) * 2.0 ** rng.integers(-12, 3, size) * rng.choice([-1, 1], size)
    smallest = rng.integers(0, 2048, size) * 2.0 ** -24
    largest = rng.choice([8184.0, -8184.0, 4093.0, 8180.0], size)
    for d in (ordinary, smallest, largest):
        c, want = q4_case(dev, counts, n, k, torch.from_numpy(d.astype(np.float16)).to(dev), seed=k)
        y = call_experts(c, out_dtype=torch.float32)
        assert torch.equal(y.double(), want)


@pytest.mark.parametrize("counts", [[5, 9, 0, 20], [17, 2, 24, 16], [300, 41], [257, 600, 3]])
@pytest.mark.parametrize("n,k", [(40, 96), (130, 416), (200, 1408), (64, 4096)])
def test_mul_mat_id_q4_sums_are_those_of_fp32(dev, counts, n, k):
    """An fp32 sum of two products a weight (the weight as two numbers) and nothing else."""
    for glu in (False, True):
        c = make_experts(dev, sum(counts), len(counts), 1, n, k, "q4_0", glu, seed=k, ids=slots_of(counts, dev))
        ref, _ = experts_reference(c)
        mag = torch.zeros(sum(counts), n * (1 + glu), dtype=torch.float64, device=dev)
        z = torch.zeros_like(mag)
        for e in range(len(counts)):
            s = torch.nonzero(c["ids"].view(-1) == e).flatten()
            mag[s] = c["x"][s].double().abs() @ c["w64"][e].abs().t()
            z[s] = c["x"][s].double() @ c["w64"][e].t()
        dz = (2 * k + 8) * 2.0 ** -24 * mag
        if glu:  # as of the 16-bit weights: |silu'| < 1.1, exp, a sum, a division and two products
            gate, up = z[:, :n], z[:, n:]
            silu = gate * torch.sigmoid(gate)
            tol = 1.1 * dz[:, :n] * up.abs() + silu.abs() * dz[:, n:] + 1.1 * dz[:, :n] * dz[:, n:] + 2.0 ** -20 * (silu * up).abs()
        else:
            tol = dz
        check_rows(call_experts(c, out_dtype=torch.float32), ref, tol)


@pytest.mark.parametrize("T", [5, 40, 1500])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("dt,bits", [("bf16", 24), ("f16", 22)])
def test_lora_rank_values_are_exact(dev, T, rank, dt, bits):
    """Rank values of 24 bits (bf16: three numbers of 8) or 22 (fp16: two of 11) come through B = 1 as they are."""
    rng = np.random.default_rng(rank)
    piece = bits // (3 if dt == "bf16" else 2)
    h = rng.integers(2 ** (bits - 1), 2 ** bits, rank)  # of one row, all of one size
    parts = [(h >> (bits - piece * (i + 1))) & (2 ** piece - 1) for i in range(bits // piece)]
    assert np.array_equal(sum(p << (bits - piece * (i + 1)) for i, p in enumerate(parts)), h)
    a = torch.zeros(1, rank, 64, dtype=torch.float64, device=dev)
    x = torch.zeros(T, 64, dtype=torch.float64, device=dev)
    for i, p in enumerate(parts):  # x a: the pieces' sum
        a[0, :, 5 + 20 * i] = torch.from_numpy(p * 2.0 ** -piece).to(dev)
        x[:, 5 + 20 * i] = 2.0 ** (-piece * i)
    want = torch.from_numpy(h * 2.0 ** -bits).to(dev)
    assert torch.equal(x.to(DT[dt]).double(), x) and torch.equal(a.to(DT[dt]).double(), a)
    assert torch.equal((x @ a[0].t()), want.expand(T, rank))
    ids = torch.zeros(T, dtype=torch.int32, device=dev)
    c = {"x": x.to(DT[dt]), "a": a.to(DT[dt]), "b": torch.eye(rank, device=dev).to(DT[dt])[None].contiguous(), "scales": None,
         "resid": torch.zeros(T, rank, device=dev), "ids": ids}
    assert torch.equal(call_lora(c).double(), want.expand(T, rank))


@pytest.mark.parametrize("T", [5, 1500])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_lora_infinite_values_of_one_sign_stay_infinite(dev, T, rank, dt):
    """Ranks between the kernel's widths: no NaN out of an infinity where the formula has none."""
    c = make_lora(dev, T, 2, rank, 64, 40, dt, "f32", seed=rank)
    c["a"], c["b"] = c["a"].abs() + 2.0 ** -6, c["b"].abs() + 2.0 ** -6
    c["ids"][:] = torch.arange(T, device=dev) % 2
    c["x"][1, 3], c["x"][2, 60] = math.inf, -math.inf
    y = call_lora(c)
    assert bool((y[1] == math.inf).all()) and bool((y[2] == -math.inf).all())
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[[1, 2]] = False
    ref, tol = lora_reference(c)
    check_rows(y[keep], ref[keep], tol[keep])


# ------------------------------------------------------------------------------ where the plans go from one launch to two
@pytest.mark.parametrize("T", [31, 32, 33, 63, 64, 65, 96, 97, 4735, 4736, 4737])
@pytest.mark.parametrize("E,top", [(5, 2), (64, 4), (64, 5), (65, 4), (300, 8), (1024, 1)])
def test_route_of_one_launch_and_of_two(dev, T, E, top):
    g = torch.Generator(device=dev).manual_seed(T + E)
    x = 2 * torch.randn(T, E, generator=g, device=dev)
    check_route(b2q.moe_route(x, top), x, None, top, "softmax", True)


@pytest.mark.parametrize("S", [511, 513, 2047, 2048, 2049, 2560, 2561, 75775, 75777])
@pytest.mark.parametrize("groups", [1, 64, 1024])
def test_group_rows_of_one_launch_and_of_two(dev, S, groups):
    ids = np.random.default_rng(S).integers(-1, groups + 1, S).astype(np.int32)
    order, offsets = b2q.group_rows(torch.from_numpy(ids).to(dev), groups)
    ro, rf = plan_reference(ids, groups)
    assert np.array_equal(order.cpu().numpy(), ro) and np.array_equal(offsets.cpu().numpy(), rf)


# --------------------------------------------------------------------------------------- requests of a larger buffer
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 0), (0, 4), (700, 600)])
def test_verify_rows_before_the_first_request_and_behind_the_last(dev, before, behind):
    """A stretch of a buffer's requests: its own rows as if it were alone, -1 in all others."""
    g = torch.Generator(device=dev).manual_seed(before)
    B, D, V = 3, 7, 90
    p = torch.softmax(2 * torch.randn(before + D + B + behind, V, generator=g, device=dev), -1)
    q = torch.softmax(2 * torch.randn(before + D + behind, V, generator=g, device=dev), -1)
    drafts = torch.randint(0, V, (before + D + behind,), generator=g, device=dev).int()
    u, v = torch.rand(before + D + behind, generator=g, device=dev), torch.rand(B, generator=g, device=dev)
    cu = torch.tensor([0, 2, 2, 7], dtype=torch.int32, device=dev)
    alone = b2q.draft_verify(p[before:before + D + B].contiguous(), q[before:before + D].contiguous(), drafts[before:before + D].contiguous(),
                             cu, u[before:before + D].contiguous(), v)
    # memory that is not -1 by chance: the allocator hands out what was just freed
    torch.full((before + D + B + behind,), 77, dtype=torch.int32, device=dev)
    accepted, tokens = b2q.draft_verify(p, q, drafts, cu + before, u, v)
    assert torch.equal(accepted, alone[0]) and torch.equal(tokens[before:before + D + B], alone[1])
    assert bool((tokens[:before] == -1).all()) and bool((tokens[before + D + B:] == -1).all())


# ------------------------------------------------------------------------- experts and adapters in one block
@pytest.mark.parametrize("counts", [[3, 2], [70, 41]])
def test_block_with_experts_and_adapters_of_the_attention(dev, counts):
    """What the block gives with both: its attention with adapters (of a block whose last linears add nothing), then the
    experts on that."""
    C, heads, D, hidden, sections, G, rank = 256, 4, 64, 512, (12, 10, 10), 3, 16
    _, weights = cb.random_block(dev, C, heads, heads, D, hidden, sections, seed=5)
    weights["fc2"] = np.zeros_like(weights["fc2"])
    g = torch.Generator(device=dev).manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    vec = {"b_qkv": 0.1 * r(3 * heads * D), "b_out": 0.1 * r(C), "b1": 0.1 * r(hidden), "b2": torch.zeros(C, device=dev),
           "gq": 1 + 0.1 * r(heads * D), "gk": 1 + 0.1 * r(heads * D)}
    freq = 1e4 ** (-torch.cat([torch.arange(n, device=dev) / n for n in sections]))
    make = lambda **kw: cb.CachedBlock(dev, weights, vec, C, heads, heads, D, hidden, sections, freq, unrounded_rows=128, **kw)  # noqa: E731
    experts, _ = cb.random_experts(dev, 6, C, 96, 2, seed=2)
    both, attention = make(experts=experts), make()
    shapes = cb.CachedBlock.shapes(C, heads, heads, D, hidden)
    pairs = {n: ((r(G, rank, shapes[n][1]) / shapes[n][1] ** 0.5).half(), (0.3 * r(G, shapes[n][0], rank) / rank ** 0.5).half())
             for n in ("qkv", "out")}
    adapters = cb.Adapters(pairs)
    ids = torch.repeat_interleave(torch.tensor([2, -1]), torch.tensor(counts)).int().to(dev)
    x = r(sum(counts), C)

    def run(block, adapters):
        cache = cb.PagedCache(dev, 1, 2, heads, D, pages=20, page_size=16, max_len=128)
        step = cache.plan(counts)
        pos = step["pos"]
        grid = torch.stack([pos, pos // 7, pos % 7]).int().contiguous()
        rows = adapters.plan(ids) if adapters else None
        return block.forward(x.clone(), cache, 0, step, grid, adapters=adapters, rows=rows)

    mid = run(attention, adapters)
    assert torch.equal(run(both, adapters), experts.forward(b2q.norm_modulate(mid), mid.clone()))
    plain = run(both, None)
    assert torch.equal(run(both, adapters)[counts[0]:], plain[counts[0]:]) and not torch.equal(run(both, adapters), plain)
