"""Rows that go by group (b2q_moe_route, b2q_group_rows, b2q_mul_mat_id, b2q_moe_combine, b2q_lora_add) against plain
64-bit arithmetic.  Tolerances: a rounding is half a step of its type, relative; an fp32 sum of n products is off by at
most (n + 8) 2^-24 of the sum of their magnitudes."""
import math

import numpy as np
import pytest
import torch

import b2q

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WT = {"f16": b2q.TYPE_F16, "bf16": b2q.TYPE_BF16, "q4_0": b2q.TYPE_Q4_0}


def half_step(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture(autouse=True)
def no_device_error(dev):
    yield
    assert b2q.device_status() == 0


# ------------------------------------------------------------------------------------------------------- the router
def route_reference(x, bias, top, scoring, renorm, scale):
    """numpy float32 logits -> ids, float64 weights."""
    key = x if bias is None else (x + bias).astype(np.float32)
    key = np.where(np.isnan(key), -np.inf, key)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :top]
    none = np.take_along_axis(key, ids, 1) == -np.inf
    ids = np.where(none, -1, ids)
    z = x.astype(np.float64)
    picked = np.take_along_axis(z, np.maximum(ids, 0), 1)
    if scoring == "sigmoid":
        w = 1 / (1 + np.exp(-picked))
    else:
        z = np.where(np.isnan(z), -np.inf, z)
        m = z.max(1, keepdims=True)
        m = np.where(m == -np.inf, 0.0, m)
        gap = lambda v: np.where(v == m, 0.0, v - m)  # noqa: E731
        w = np.exp(gap(picked)) / np.maximum(np.exp(gap(z)).sum(1, keepdims=True), 1e-300)
    w = np.where(none, 0.0, w)
    if renorm:
        s = w.sum(1, keepdims=True)
        w = np.where(s > 0, w / np.where(s > 0, s, 1), 0.0)
    return ids, w * scale


def plan_reference(ids, groups):
    flat = np.asarray(ids).reshape(-1)
    flat = np.where((flat < 0) | (flat >= groups), groups, flat)
    counts = np.bincount(flat, minlength=groups + 1)
    return np.argsort(flat, kind="stable"), np.concatenate([[0], np.cumsum(counts[:groups])])


def check_route(got, x, bias, top, scoring, renorm, scale=1.0):
    ids, weights, order, offsets = got
    E = x.shape[1]
    b = None if bias is None else bias.cpu().numpy()
    with np.errstate(all="ignore"):
        ri, rw = route_reference(x.float().cpu().numpy(), b, top, scoring, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), ri)
    # exp of a difference (2^-24 of its size, at most 100), the division and sums of at most E terms
    tol = (E + 120) * 2.0 ** -24
    w = weights.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(w - rw) <= tol * np.abs(rw) + 1e-37)
    ro, rf = plan_reference(ri, E)
    assert np.array_equal(order.cpu().numpy(), ro) and np.array_equal(offsets.cpu().numpy(), rf)


@pytest.mark.parametrize("T,E,top", [(1, 1, 1), (1, 64, 6), (12, 64, 6), (3, 7, 7), (33, 33, 4), (128, 16, 16), (700, 160, 8),
                                     (4097, 31, 3), (513, 1024, 32), (20000, 8, 2), (9, 300, 32)])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_route(dev, T, E, top, ty):
    g = torch.Generator(device=dev).manual_seed(T + E)
    x = (2 * torch.randn(T, E, generator=g, device=dev)).to(DT[ty])
    bias = 0.5 * torch.randn(E, generator=g, device=dev)
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            for b in (None, bias):
                check_route(b2q.moe_route(x, top, bias=b, scoring=scoring, renorm=renorm, scale=1.5), x, b, top, scoring,
                            renorm, 1.5)


@pytest.mark.parametrize("T", [5, 1500])
def test_route_ties_zeros_and_masked_experts(dev, T):
    """Equal logits, zeros of both signs, infinities, NaN, rows with fewer experts than choices and rows with none."""
    E, top = 40, 6
    rng = np.random.default_rng(5)
    x = rng.integers(-2, 3, (T, E)).astype(np.float32)
    x[x == 0] *= rng.choice([-1.0, 1.0], int((x == 0).sum()))
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = -np.inf
    x[3, [7, 30]] = [1.0, 2.0]
    x[4, :] = -np.inf
    x[4, 11] = -3e38
    x[0, ::3] = np.nan
    x[T // 2, 5] = -np.inf
    xd = torch.from_numpy(x).to(dev)
    bias = torch.zeros(E, device=dev)
    bias[9] = -math.inf
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            for b in (None, bias):
                check_route(b2q.moe_route(xd, top, bias=b, scoring=scoring, renorm=renorm), xd, b, top, scoring, renorm)


def test_route_infinite_logits_share_the_weight(dev):
    x = torch.zeros(2, 8, device=dev)
    x[0, [2, 5]] = math.inf
    x[1, 3] = math.inf
    ids, w, _, _ = b2q.moe_route(x, 3)
    assert ids.tolist() == [[2, 5, 0], [3, 0, 1]]
    assert w.tolist() == [[0.5, 0.5, 0.0], [1.0, 0.0, 0.0]]


def test_route_row_strides(dev):
    wide = torch.randn(300, 100, device=dev)
    x = wide[:, 3:53]
    check_route(b2q.moe_route(x, 4), x, None, 4, "softmax", True)


def test_route_of_no_tokens(dev):
    ids, w, order, offsets = b2q.moe_route(torch.empty(0, 12, device=dev), 3)
    assert ids.shape == (0, 3) and w.shape == (0, 3) and order.numel() == 0 and offsets.tolist() == [0] * 13


@pytest.mark.parametrize("S,groups", [(1, 1), (5, 1000), (2048, 64), (2049, 64), (30000, 3), (100003, 1024), (400000, 17)])
def test_group_rows(dev, S, groups):
    rng = np.random.default_rng(S)
    ids = rng.integers(-2, groups + 2, S).astype(np.int32)
    ids[S // 3:S // 2] = groups // 2  # a long run of one group
    order, offsets = b2q.group_rows(torch.from_numpy(ids).to(dev), groups)
    ro, rf = plan_reference(ids, groups)
    assert np.array_equal(order.cpu().numpy(), ro) and np.array_equal(offsets.cpu().numpy(), rf)


def test_group_rows_of_nothing(dev):
    order, offsets = b2q.group_rows(torch.empty(0, dtype=torch.int32, device=dev), 5)
    assert order.numel() == 0 and offsets.tolist() == [0] * 6
    order, offsets = b2q.group_rows(torch.full((3000,), -1, dtype=torch.int32, device=dev), 5)
    assert offsets.tolist() == [0] * 6 and order.tolist() == list(range(3000))


# ----------------------------------------------------------------------------------------------- the experts' products
def q4_blocks(rows, k, g, dev, scale=None):
    """Q4_0 rows and their values in 64 bits."""
    raw = torch.randint(0, 256, (rows, k // 32, 18), dtype=torch.uint8, generator=g, device=dev)
    d = ((0.3 / math.sqrt(k) if scale is None else scale) * (1 + torch.rand(rows, k // 32, 1, generator=g, device=dev))).half()
    raw[:, :, :2] = d.view(torch.uint8)
    codes = torch.cat([raw[:, :, 2:] & 15, raw[:, :, 2:] >> 4], -1).double() - 8
    return raw.view(rows, -1), (codes * d.double()).view(rows, k)


def make_experts(dev, T, E, top, n, k, wname, glu=False, per_row=None, seed=0, ids=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = 2 * n if glu else n
    dt = DT["f16" if wname == "q4_0" else wname]
    if ids is None:
        ids = torch.stack([torch.randperm(E, generator=g, device=dev)[:top] for _ in range(T)]).int()
        ids[torch.rand(T, top, generator=g, device=dev) < 0.1] = -1
    per_row = top if per_row is None else per_row
    x = torch.randn(-(-T * top // per_row), k, generator=g, device=dev).to(dt)
    if wname == "q4_0":
        raw, w64 = q4_blocks(E * rows, k, g, dev)
        w = b2q.weight_pack_q4_0(raw, k)
    else:
        w = (torch.randn(E * rows, k, generator=g, device=dev) / math.sqrt(k)).to(dt)
        w64 = w.double()
        w = w.view(E, rows, k)
    return {"x": x, "w": w, "w64": w64.view(E, rows, k), "ids": ids, "n": n, "k": k, "per_row": per_row, "glu": glu,
            "wtype": WT[wname], "E": E, "dt": dt}


def experts_reference(c, bias=None):
    """(result, tolerance before the last rounding) per slot, in 64 bits."""
    ids = c["ids"].reshape(-1).long()
    S, n = ids.numel(), c["n"]
    y = torch.zeros(S, n, dtype=torch.float64, device=ids.device)
    tol = torch.zeros_like(y)
    sums = (c["k"] + 8) * 2.0 ** -24
    for e in range(c["E"]):
        s = torch.nonzero(ids == e).flatten()
        if not s.numel():
            continue
        x, w = c["x"][s // c["per_row"]].double(), c["w64"][e]
        z, mag = x @ w.t(), x.abs() @ w.abs().t()
        # a 4-bit weight's value may be rounded to fp16 (half a step, or half the smallest number)
        dz = sums * mag + (2.0 ** -11 * mag + 2.0 ** -25 * x.abs().sum(1, keepdim=True) if c["wtype"] == b2q.TYPE_Q4_0 else 0)
        if bias is not None:
            z = z + bias.view(c["E"], -1)[e].double()
            dz = dz + 2.0 ** -24 * z.abs()
        if c["glu"]:
            gate, up = z[:, :n], z[:, n:]
            silu = gate * torch.sigmoid(gate)
            y[s] = silu * up
            # |silu'| < 1.1; exp of a number up to 2^7, a sum, a division and two products
            tol[s] = 1.1 * dz[:, :n] * up.abs() + silu.abs() * dz[:, n:] + 1.1 * dz[:, :n] * dz[:, n:] \
                + 2.0 ** -20 * (silu * up).abs()
        else:
            y[s], tol[s] = z, dz
    return y, tol


def call_experts(c, order=None, offsets=None, **kw):
    if order is None:
        order, offsets = b2q.group_rows(c["ids"].contiguous(), c["E"])
    return b2q.mul_mat_id(c["wtype"], c["w"], c["n"], c["k"], c["x"], order, offsets, per_row=c["per_row"], glu=c["glu"], **kw)


def check_rows(y, ref, tol):
    err = (y.double() - ref).abs()
    assert bool((err <= tol + half_step(y.dtype) * (ref.abs() + tol) + 1e-37 + (2.0 ** -25 if y.dtype is torch.float16 else 0)).all()), \
        float((err / (tol + half_step(y.dtype) * ref.abs() + 1e-30)).max())


@pytest.mark.parametrize("wname", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("T,E,top,n,k", [(1, 1, 1, 1, 32), (1, 8, 2, 64, 64), (2, 64, 6, 96, 256), (7, 5, 3, 33, 96),
                                         (40, 16, 4, 200, 416), (129, 3, 2, 130, 1024), (300, 2, 1, 257, 160),
                                         (700, 4, 3, 128, 2048), (1100, 1, 1, 300, 64)])
def test_mul_mat_id(dev, wname, glu, T, E, top, n, k):
    c = make_experts(dev, T, E, top, n, k, wname, glu, seed=T)
    g = torch.Generator(device=dev).manual_seed(1)
    bias = torch.randn(E * n * (1 + glu), generator=g, device=dev)
    for b in (None, bias):
        ref, tol = experts_reference(c, b)
        for out in (None, torch.float32):
            y = call_experts(c, bias=b, out_dtype=out)
            assert y.dtype is (out or c["dt"])
            check_rows(y, ref, tol)
            none = (c["ids"].reshape(-1) < 0)
            assert bool((y[none] == 0).all())


@pytest.mark.parametrize("wname,k", [("f16", 8), ("bf16", 24), ("f16", 1000), ("bf16", 72), ("q4_0", 32), ("q4_0", 1376)])
@pytest.mark.parametrize("n", [1, 31, 131])
def test_mul_mat_id_odd_sizes(dev, wname, k, n):
    for glu in (False, True):
        c = make_experts(dev, 50, 6, 2, n, k, wname, glu, seed=n + k)
        ref, tol = experts_reference(c)
        check_rows(call_experts(c), ref, tol)


@pytest.mark.parametrize("per_row", [1, 2, 3, 6])
def test_mul_mat_id_rows_of_x(dev, per_row):
    c = make_experts(dev, 60, 9, 6, 40, 128, "bf16", per_row=per_row, seed=3)
    ref, tol = experts_reference(c)
    check_rows(call_experts(c), ref, tol)


@pytest.mark.parametrize("wname", ["f16", "q4_0"])
@pytest.mark.parametrize("counts", [[0, 0, 500, 0], [1, 0, 0, 0], [0, 0, 0, 0], [255, 1, 256, 257], [31, 32, 33, 0],
                                    [511, 513, 1, 16]])
def test_mul_mat_id_uneven_groups(dev, wname, counts):
    ids = torch.cat([torch.full((n,), e, dtype=torch.int32) for e, n in enumerate(counts)] + [torch.full((9,), -1, dtype=torch.int32)])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))].view(-1, 1).to(dev)
    for glu in (False, True):
        c = make_experts(dev, ids.numel(), 4, 1, 150, 192, wname, glu, ids=ids)
        ref, tol = experts_reference(c)
        check_rows(call_experts(c), ref, tol)


def test_mul_mat_id_strides(dev):
    """Rows of x, of the weight and of y, and experts, further apart than they are long."""
    c = make_experts(dev, 90, 5, 2, 72, 64, "f16", seed=4)
    ref, tol = experts_reference(c)
    wide = torch.full((5, 80, 88), math.nan, dtype=torch.float16, device=dev)
    wide[:, :72, :64] = c["w"]
    x = torch.full((90, 104), math.nan, dtype=torch.float16, device=dev)
    x[:, :64] = c["x"]
    out = torch.full((180, 99), 7.0, dtype=torch.float16, device=dev)
    c["w"], c["x"] = wide[:, :72, :64], x[:, :64]
    y = call_experts(c, out=out[:, :72])
    assert y.data_ptr() == out.data_ptr()
    check_rows(out[:, :72], ref, tol)
    assert bool((out[:, 72:] == 7.0).all())


@pytest.mark.parametrize("wname", ["f16", "q4_0"])
@pytest.mark.parametrize("T", [3, 700])
def test_results_beside_their_operands(dev, wname, T):
    """Columns of one table are disjoint although their memory is not."""
    c = make_experts(dev, T, 4, 1, 64, 64, wname, seed=5)
    ref, tol = experts_reference(c)
    table = torch.full((T, 144), 7.0, dtype=torch.float16, device=dev)
    table[:, :64] = c["x"]
    call_experts(dict(c, x=table[:, :64]), out=table[:, 72:136])
    check_rows(table[:, 72:136], ref, tol)
    assert torch.equal(table[:, :64], c["x"]) and bool((table[:, 64:72] == 7.0).all()) and bool((table[:, 136:] == 7.0).all())
    with pytest.raises(RuntimeError):
        call_experts(dict(c, x=table[:, :64]), out=table[:, 56:120])
    c = make_lora(dev, T, 4, 16, 64, 64, "f16", "f16", seed=5)
    ref, tol = lora_reference(c)
    table[:, :64], table[:, 72:136] = c["x"], c["resid"]
    y = table[:, 72:136]
    call_lora(dict(c, x=table[:, :64], resid=y), out=y)
    check_rows(y, ref, tol)
    assert torch.equal(table[:, :64], c["x"]) and bool((table[:, 64:72] == 7.0).all()) and bool((table[:, 136:] == 7.0).all())
    with pytest.raises(RuntimeError):
        call_lora(dict(c, x=table[:, :64]), out=table[:, 56:120])


@pytest.mark.parametrize("layout", ["padded", "rows first", "one expert"])
def test_mul_mat_id_glu_strides(dev, layout):
    """Gate and up rows of experts that lie an odd number of rows apart, of row-major stacks, and of one expert."""
    E = 1 if layout == "one expert" else 5
    c = make_experts(dev, 90, E, 1, 36, 64, "bf16", glu=True, seed=4)
    ref, tol = experts_reference(c)
    if layout == "rows first":
        wide = torch.full((72, E, 64), math.nan, dtype=torch.bfloat16, device=dev)
        wide.copy_(c["w"].transpose(0, 1))
        c["w"] = wide.transpose(0, 1)
    else:
        wide = torch.full((E, 75, 72), math.nan, dtype=torch.bfloat16, device=dev)
        wide[:, :72, :64] = c["w"]
        c["w"] = wide[:, :72, :64]
    check_rows(call_experts(c), ref, tol)


@pytest.mark.parametrize("k,T", [(4096, 3), (4096, 150), (6144, 5), (4480, 40)])
def test_mul_mat_id_q4_long_rows(dev, k, T):
    """Rows that fill the few-row kernel's shared memory (8 slots at a time), and rows that do not fit it."""
    for glu in (False, True):
        c = make_experts(dev, T, 4, 2, 40, k, "q4_0", glu, seed=k)
        ref, tol = experts_reference(c)
        check_rows(call_experts(c), ref, tol)


def test_mul_mat_id_inputs_of_other_rows_do_not_reach_a_row(dev):
    """A row of NaN and one of infinities among the rows of one expert, and an expert of NaN."""
    c = make_experts(dev, 200, 3, 1, 64, 128, "bf16", seed=5, ids=torch.zeros(200, 1, dtype=torch.int32, device=dev))
    c["ids"][150:] = 2
    c["w"] = c["w"].clone()
    c["w"][1] = math.nan
    ref, tol = experts_reference(c)
    clean = call_experts(c)
    check_rows(clean, ref, tol)
    c["x"][17] = math.nan
    c["x"][160] = math.inf
    y = call_experts(c)
    keep = torch.ones(200, dtype=torch.bool, device=dev)
    keep[[17, 160]] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(torch.isnan(y[17]).all())


def test_mul_mat_id_with_a_broken_plan_stays_inside(dev):
    """Slots and offsets outside the plan are left out; rows that the plan does name are right."""
    c = make_experts(dev, 64, 4, 1, 40, 64, "f16", seed=6)
    order, offsets = b2q.group_rows(c["ids"].contiguous(), 4)
    ref, tol = experts_reference(c)
    bad = order.clone()
    bad[[0, 20]] = torch.tensor([-5, 1 << 29], dtype=torch.int32, device=dev)
    out = torch.full((64, 40), 5.0, dtype=torch.float16, device=dev)
    call_experts(c, bad, offsets, out=out)
    missing = order[[0, 20]].long()
    assert bool((out[missing] == 5.0).all())
    keep = torch.ones(64, dtype=torch.bool, device=dev)
    keep[missing] = False
    check_rows(out[keep], ref[keep], tol[keep])
    wild = torch.tensor([-9, 1 << 30, 3, -1, 1 << 30], dtype=torch.int32, device=dev)
    call_experts(c, order, wild)
    torch.cuda.synchronize()


def test_mul_mat_id_repeats_bit_for_bit(dev):
    c = make_experts(dev, 500, 7, 3, 160, 512, "bf16", glu=True, seed=8)
    order, offsets = b2q.group_rows(c["ids"].contiguous(), 7)
    first = call_experts(c, order, offsets)
    for _ in range(3):
        assert torch.equal(call_experts(c, order, offsets), first)


@pytest.mark.parametrize("T,top,n", [(1, 1, 1), (3, 2, 7), (40, 6, 200), (513, 4, 1033), (2, 33, 64)])
@pytest.mark.parametrize("yt,ot", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f16")])
def test_combine(dev, T, top, n, yt, ot):
    g = torch.Generator(device=dev).manual_seed(T * n)
    y = torch.randn(T * top, n, generator=g, device=dev).to(DT[yt])
    w = torch.rand(T, top, generator=g, device=dev)
    ids = torch.randint(-1, 3, (T, top), generator=g, device=dev).int()
    y[ids.view(-1) < 0] = math.nan  # not read
    resid = torch.randn(T, n, generator=g, device=dev).to(DT[ot])
    live = (ids >= 0).double()
    terms = torch.nan_to_num(y.double()).view(T, top, n) * (w.double() * live)[:, :, None]
    for r in (None, resid):
        ref = terms.sum(1) + (0 if r is None else r.double())
        mag = terms.abs().sum(1) + (0 if r is None else r.double().abs())
        out = b2q.moe_combine(y, w, ids, resid=r, out_dtype=DT[ot])
        check_rows(out, ref, (top + 2) * 2.0 ** -24 * mag)
    mine = resid.clone()
    assert b2q.moe_combine(y, w, ids, resid=mine, out=mine) is mine
    assert torch.equal(mine, b2q.moe_combine(y, w, ids, resid=resid))


# -------------------------------------------------------------------------------------------------------- the adapters
def make_lora(dev, T, G, rank, k, n, dt, out, seed=0, ids=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    if ids is None:
        ids = torch.randint(-1, G, (T,), generator=g, device=dev).int()
    return {"x": r(T, k).to(DT[dt]), "a": (r(G, rank, k) / math.sqrt(k)).to(DT[dt]), "b": (r(G, n, rank) / math.sqrt(rank)).to(DT[dt]),
            "scales": 0.5 + torch.rand(G, generator=g, device=dev), "resid": r(T, n).to(DT[out]), "ids": ids}


def lora_reference(c, scales=True):
    k, rank = c["x"].shape[1], c["a"].shape[1]
    y, tol = c["resid"].double(), torch.zeros(c["resid"].shape, dtype=torch.float64, device=c["x"].device)
    for i in range(c["a"].shape[0]):
        t = torch.nonzero(c["ids"] == i).flatten()
        if not t.numel():
            continue
        x, a, b = c["x"][t].double(), c["a"][i].double(), c["b"][i].double()
        s = float(c["scales"][i]) if scales else 1.0
        h, mag = x @ a.t() * s, x.abs() @ a.abs().t() * s
        # the rank values: an fp32 sum, the scale, and two 16-bit numbers (half a step of half a step of the row's largest)
        dh = (k + 10) * 2.0 ** -24 * mag + 2.0 ** -17 * h.abs().amax(1, keepdim=True)
        d = h @ b.t()
        y[t] += d
        tol[t] = dh @ b.abs().t() + (2 * rank + 8) * 2.0 ** -24 * (h.abs() @ b.abs().t()) + 2.0 ** -24 * (y[t].abs() + d.abs())
    return y, tol


def call_lora(c, **kw):
    order, offsets = b2q.group_rows(c["ids"], c["a"].shape[0])
    return b2q.lora_add(c["resid"], c["x"], c["a"], c["b"], c["scales"], order, offsets, **kw)


@pytest.mark.parametrize("dt,out", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,G,rank,k,n", [(1, 1, 8, 8, 1), (1, 3, 16, 64, 64), (5, 40, 8, 1000, 33), (32, 24, 16, 4096, 520),
                                          (64, 2, 128, 256, 130), (300, 3, 64, 520, 1030), (1000, 5, 24, 136, 77),
                                          (2500, 2, 40, 72, 264), (70, 70, 104, 2048, 16), (1700, 3, 16, 256, 129),
                                          (1800, 9, 64, 1032, 200), (1600, 2, 128, 136, 321), (3000, 40, 32, 64, 96)])
def test_lora(dev, dt, out, T, G, rank, k, n):
    c = make_lora(dev, T, G, rank, k, n, dt, out, seed=T + n)
    ref, tol = lora_reference(c)
    y = call_lora(c)
    check_rows(y, ref, tol)
    none = c["ids"] < 0
    assert torch.equal(y[none], c["resid"][none])
    mine = c["resid"].clone()
    c2 = dict(c, resid=mine)
    assert call_lora(c2, out=mine) is mine and torch.equal(mine, y)


@pytest.mark.parametrize("k", [264, 520, 1032, 2056])
@pytest.mark.parametrize("T,G,rank,n", [(830, 2, 64, 130), (830, 5, 8, 64), (400, 3, 72, 256), (7000, 2, 40, 72)])
def test_lora_parts_of_k(dev, k, T, G, rank, n):
    """Two launches, K shared out over one to eight blocks, some of which may have nothing."""
    c = make_lora(dev, T, G, rank, k, n, "f16", "f32", seed=6)
    ref, tol = lora_reference(c)
    y = call_lora(c)
    check_rows(y, ref, tol)
    assert torch.equal(y, call_lora(c))


@pytest.mark.parametrize("T", [90, 1900])
def test_lora_without_scales_and_with_strides(dev, T):
    c = make_lora(dev, T, 4, 16, 128, 100, "f16", "f32", seed=2)
    c["scales"] = None
    ref, tol = lora_reference(c, scales=False)
    wide = torch.zeros(T, 160, dtype=torch.float16, device=dev)
    wide[:, :128] = c["x"]
    res = torch.zeros(T, 111, device=dev)
    res[:, 3:103] = c["resid"]
    out = torch.full((T, 107), 7.0, device=dev)
    y = call_lora(dict(c, x=wide[:, :128], resid=res[:, 3:103]), out=out[:, 1:101])
    check_rows(y, ref, tol)
    assert bool((out[:, 0] == 7.0).all()) and bool((out[:, 101:] == 7.0).all())


@pytest.mark.parametrize("T", [20, 400, 2000])
@pytest.mark.parametrize("big", [3e4, 1e-6])
def test_lora_rank_values_beyond_16_bits(dev, T, big):
    """A x that overflows fp16, or lies among its smallest numbers, still counts."""
    c = make_lora(dev, T, 3, 16, 64, 50, "f16", "f32", seed=3)
    c["x"] = (c["x"] * min(big, 1000)).clamp(-6e4, 6e4)
    c["a"] = (c["a"] * (80 if big > 1 else 1e-2)).half()
    c["b"] = (c["b"] * 1e-3).half()
    c["resid"].zero_()
    ref, tol = lora_reference(c)
    assert big < 1 or float((c["x"].double() @ c["a"][0].double().t()).abs().max()) > 65504
    check_rows(call_lora(c), ref, tol)


@pytest.mark.parametrize("T", [200, 2200])
def test_lora_non_finite_rows_stay_alone(dev, T):
    c = make_lora(dev, T, 2, 16, 128, 64, "bf16", "f32", seed=4)
    clean = call_lora(c)
    c["x"][31] = math.nan
    c["ids"][31] = 0
    c["x"][100] = math.inf
    c["ids"][100] = 1
    order, offsets = b2q.group_rows(c["ids"], 2)
    y = call_lora(c)
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[[31, 100]] = False
    ref, tol = lora_reference(c)
    check_rows(y[keep], ref[keep], tol[keep])
    assert bool(torch.isnan(y[31]).all())
    assert clean.shape == y.shape


@pytest.mark.parametrize("T", [64, 2000])
def test_lora_with_a_broken_plan_stays_inside(dev, T):
    c = make_lora(dev, T, 4, 8, 64, 40, "f16", "f32", seed=6)
    order, offsets = b2q.group_rows(c["ids"], 4)
    bad = order.clone()
    bad[[1, 30]] = torch.tensor([-5, 1 << 29], dtype=torch.int32, device=dev)
    for o, f in ((bad, offsets), (order, torch.tensor([-9, 1 << 30, 3, -1, 1 << 30], dtype=torch.int32, device=dev))):
        b2q.lora_add(c["resid"], c["x"], c["a"], c["b"], c["scales"], o, f)
    torch.cuda.synchronize()


# ----------------------------------------------------------------------------------------------------- far apart rows
def test_rows_further_apart_than_32_bits_count(dev):
    """Rows of x, y, resid and probabilities whose offsets pass 2^32 values: the results of the same rows close together."""
    far = 1 << 27  # 40 rows: 5.4e9 values of 2 bytes, in two buffers
    one, two = (torch.empty(39 * far + 256, dtype=torch.float16, device=dev) for _ in range(2))

    def spread(buf, t):
        v = buf.as_strided((t.shape[0], t.shape[1]), (far, 1))
        v.copy_(t)
        return v

    c = make_experts(dev, 40, 4, 1, 96, 64, "f16", seed=1, ids=torch.arange(40, dtype=torch.int32, device=dev).view(40, 1) % 4)
    want = call_experts(c)
    y = two.as_strided((40, 96), (far, 1))
    got = call_experts(dict(c, x=spread(one, c["x"])), out=y)
    assert torch.equal(got, want)
    q = make_experts(dev, 40, 4, 1, 96, 64, "q4_0", seed=1, ids=c["ids"])
    want = call_experts(q)
    assert torch.equal(call_experts(dict(q, x=spread(one, q["x"])), out=y), want)
    share = torch.rand(20, 2, device=dev)
    want = b2q.moe_combine(want, share)
    assert torch.equal(b2q.moe_combine(y, share), want)
    for G in (4, 1):
        lo = make_lora(dev, 40, G, 16, 64, 80, "f16", "f16", seed=2)
        want = call_lora(lo)
        assert torch.equal(call_lora(dict(lo, x=spread(one, lo["x"]), resid=spread(two, lo["resid"])), out=two.as_strided((40, 80), (far, 1))), want)
    p = torch.softmax(2 * torch.randn(30, 200, device=dev), -1).half()
    cu = torch.arange(0, 21, 2, dtype=torch.int32, device=dev)
    drafts = p[:20].argmax(1).int()
    u, v = torch.rand(20, device=dev), torch.rand(10, device=dev)
    a, b = b2q.draft_verify(p, p[:20].contiguous(), drafts, cu, u, v)
    a2, b2 = b2q.draft_verify(spread(one, p), spread(two, p[:20]), drafts, cu, u, v)
    assert torch.equal(a, a2) and torch.equal(b, b2)
    logits = torch.randn(40, 50, device=dev).half()
    assert torch.equal(b2q.moe_route(logits, 4)[0], b2q.moe_route(spread(one, logits), 4)[0])


# ------------------------------------------------------------------------------------------- together, and in a graph
def test_an_expert_layer_in_a_graph_on_its_own_stream(dev):
    """Router, both products and the join, captured once and replayed on new inputs; two graphs side by side."""
    T, E, top, C, F = 50, 12, 3, 128, 96
    g = torch.Generator(device=dev).manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    wr, w1, w2 = r(E, C) / 8, (r(E, 2 * F, C) / 11).half(), (r(E, C, F) / 10).half()

    def layer(x):
        h = x.half()
        ids, share, order, offsets = b2q.moe_route(x @ wr.t(), top)
        y = b2q.mul_mat_id(b2q.TYPE_F16, w1, F, C, h, order, offsets, per_row=top, glu=True)
        z = b2q.mul_mat_id(b2q.TYPE_F16, w2, C, F, y, order, offsets, out_dtype=torch.float32)
        return b2q.moe_combine(z, share, ids, resid=x)

    xs = [r(T, C) for _ in range(2)]
    layer(xs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append(layer(x))
        graphs.append((graph, s))
    torch.cuda.synchronize()
    for _ in range(3):
        for x in xs:
            x.copy_(r(T, C))
        want = [layer(x) for x in xs]
        torch.cuda.synchronize()
        for graph, s in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_on_a_given_stream(dev):
    c = make_experts(dev, 200, 5, 2, 64, 256, "f16", seed=11)
    lo = make_lora(dev, 200, 5, 16, 256, 64, "f16", "f32", seed=11)
    want, want_lo = call_experts(c), call_lora(lo)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    order, offsets = b2q.group_rows(c["ids"].contiguous(), 5, stream=s)
    y = call_experts(c, order, offsets, stream=s)
    o2, f2 = b2q.group_rows(lo["ids"], 5, stream=s)
    z = b2q.lora_add(lo["resid"], lo["x"], lo["a"], lo["b"], lo["scales"], o2, f2, stream=s)
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(z, want_lo)


@pytest.mark.parametrize("T", [30, 2000])
def test_calls_that_follow_one_another_wait_for_one_another(dev, T):
    """Buffers written and read by neighbouring calls (a launch may begin while the one before it ends): 60 rounds of
    products, adapters and joins over the same rows give, bit for bit, what they give one by one."""
    E, top, C, F, G = 6, 2, 128, 96, 3
    g = torch.Generator(device=dev).manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    w1, w2 = (r(E, 2 * F, C) / 11).bfloat16(), (r(E, C, F) / 10).bfloat16()
    a, b, ids = (r(G, 16, C) / 11).bfloat16(), (0.3 * r(G, C, 16) / 4).bfloat16(), torch.randint(-1, G, (T,), generator=g, device=dev).int()
    rows = b2q.group_rows(ids, G)
    x = r(T, C)
    z, y = torch.empty(T * top, F, dtype=torch.bfloat16, device=dev), torch.empty(T * top, C, device=dev)

    def round_(x, wait):
        h = (x * torch.rsqrt(x.square().mean(1, keepdim=True))).bfloat16()
        wait()
        choice, share, order, offsets = b2q.moe_route(h[:, :E], top)
        wait()
        b2q.mul_mat_id(b2q.TYPE_BF16, w1, F, C, h, order, offsets, per_row=top, glu=True, out=z)
        wait()
        b2q.mul_mat_id(b2q.TYPE_BF16, w2, C, F, z, order, offsets, out=y)
        wait()
        b2q.moe_combine(y, share, choice, resid=x, out=x)
        wait()
        b2q.lora_add(x, h, a, b, None, *rows, out=x)
        wait()

    slow = x.clone()
    for _ in range(60):
        round_(slow, torch.cuda.synchronize)
    fast = x.clone()
    for _ in range(60):
        round_(fast, lambda: None)
    assert torch.equal(fast, slow) and bool(torch.isfinite(fast).all())
