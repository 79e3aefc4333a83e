"""The few-token product with 4-bit weights (b2q_mul_vec) against 64-bit
products with the oracle's dequantized weights."""
import numpy as np
import pytest
import torch

import b2q

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(dev, wtype, n, k, seed):
    """Random blocks (every code and scale value occurs), the packed weight, the
    fp64 weight, and fp64 magnitudes (for Q4_K: of its two terms)."""
    rng = np.random.default_rng(seed)
    if wtype == b2q.TYPE_Q4_0:
        raw = rng.integers(0, 256, (n, k // 32, 18), dtype=np.uint8)
        d = (rng.standard_normal((n, k // 32)) * 0.05).astype(np.float16)
        raw[:, :, :2] = d[..., None].view(np.uint8)
        lo, hi = raw[:, :, 2:] & 15, raw[:, :, 2:] >> 4
        w = np.concatenate([lo, hi], -1).astype(np.float64) - 8
        w = (w * d.astype(np.float64)[..., None]).reshape(n, k)
        mag = np.abs(w)
        rawt = torch.from_numpy(raw.reshape(n, -1)).to(dev)
        packed = b2q.weight_pack_q4_0(rawt, k)
    else:
        raw = rng.integers(0, 256, (n, k // 256, 144), dtype=np.uint8)
        d = (rng.standard_normal((n, k // 256, 2)) * 0.002).astype(np.float16)
        raw[:, :, :4] = d.view(np.uint8).reshape(n, k // 256, 4)
        w = np.empty((n, k // 256, 8, 32))
        mag = np.empty_like(w)
        for j in range(8):
            if j < 4:
                sc, mn = raw[:, :, 4 + j] & 63, raw[:, :, 8 + j] & 63
            else:
                sc = (raw[:, :, 8 + j] & 15) | ((raw[:, :, j] >> 6) << 4)
                mn = (raw[:, :, 8 + j] >> 4) | ((raw[:, :, 4 + j] >> 6) << 4)
            q = raw[:, :, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
            q = (q >> 4) if j % 2 else (q & 15)
            a = (d[:, :, 0].astype(np.float64) * sc)[..., None] * q
            b = (d[:, :, 1].astype(np.float64) * mn)[..., None]
            w[:, :, j] = a - b
            mag[:, :, j] = np.abs(a) + np.abs(b)
        w, mag = w.reshape(n, k), mag.reshape(n, k)
        rawt = torch.from_numpy(raw.reshape(n, -1)).to(dev)
        packed = b2q.weight_pack(b2q.TYPE_Q4_K, rawt, k)
    return rawt, packed, torch.from_numpy(w).to(dev), torch.from_numpy(mag).to(dev)


def bound(x, mag, k):
    """Error bound per output: every activation may be held to 2^-23 of its 32-value block's
    largest magnitude, and k / 32 fp32 block sums add up with a random walk of roundings."""
    xd = x.double().abs()
    amax = xd.view(x.shape[0], k // 32, 32).amax(-1).repeat_interleave(32, 1)
    return (8 + (k / 32) ** 0.5) * 2.0 ** -24 * (amax @ mag.t())


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
@pytest.mark.parametrize("n,k,m,xt", [
    (1, 256, 1, "f32"), (7, 256, 8, "f16"), (16, 512, 2, "bf16"), (33, 1024, 3, "f32"), (130, 2304, 4, "f32"),
    (1024, 1024, 1, "f32"), (4097, 768, 5, "f16"), (6144, 1024, 1, "bf16"), (1000, 8192, 6, "f32"),
    (515, 12544, 7, "bf16"), (257, 16384, 8, "f32"), (20011, 512, 8, "bf16"), (40000, 256, 1, "f16"),
])
def test_mul_vec(dev, wtype, n, k, m, xt):
    _, packed, w, mag = make(dev, wtype, n, k, n + k)
    g = torch.Generator(device=dev).manual_seed(m)
    x = torch.randn(m, k, generator=g, device=dev).to(DT[xt])
    y = b2q.mul_vec(wtype, packed, n, k, x)
    assert bool(((y.double() - x.double() @ w.t()).abs() <= bound(x, mag, k)).all())


@pytest.mark.parametrize("k", [32, 64, 96, 160, 288, 544, 1056, 4128, 16352])
@pytest.mark.parametrize("m,xt", [(1, "f32"), (3, "f16"), (8, "f32")])
def test_q4_0_odd_block_counts(dev, k, m, xt):
    n = 53
    _, packed, w, mag = make(dev, b2q.TYPE_Q4_0, n, k, k)
    x = (torch.randn(m, k, generator=torch.Generator(device=dev).manual_seed(k), device=dev) * 3).to(DT[xt])
    y = b2q.mul_vec(b2q.TYPE_Q4_0, packed, n, k, x)
    assert bool(((y.double() - x.double() @ w.t()).abs() <= bound(x, mag, k)).all())


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
def test_bias_gate_residual_strides(dev, wtype):
    n, k, m = 200, 1280, 5
    _, packed, w, mag = make(dev, wtype, n, k, 3)
    wide = torch.randn(m, k + 40, device=dev)
    x = wide[:, 7:7 + k]  # rows aligned to 4 bytes only
    bias, gate = torch.randn(n, device=dev), torch.randn(n, device=dev)
    resid = torch.randn(m, n + 3, device=dev)
    ref = x.double() @ w.t()
    tol = bound(x.contiguous(), mag, k)
    out = torch.full((m, n + 9), 5.0, device=dev)
    b2q.mul_vec(wtype, packed, n, k, x, bias=bias, out=out[:, :n])
    r1 = ref + bias.double()
    assert bool(((out[:, :n].double() - r1).abs() <= tol + 2.0 ** -23 * r1.abs()).all())
    assert bool((out[:, n:] == 5.0).all())
    base = resid[:, :n].clone()
    b2q.mul_vec(wtype, packed, n, k, x, bias=bias, gate=gate, resid=resid[:, :n], out=resid[:, :n])
    r2 = base.double() + gate.double() * r1
    lim = tol * gate.double().abs() + 2.0 ** -22 * ((gate.double() * r1).abs() + r2.abs())
    assert bool(((resid[:, :n].double() - r2).abs() <= lim).all())
    y = b2q.mul_vec(wtype, packed, n, k, x, resid=base)
    r3 = base.double() + ref
    assert bool(((y.double() - r3).abs() <= tol + 2.0 ** -23 * (r3.abs() + ref.abs())).all())


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
def test_wide_range_of_activations(dev, wtype):
    """Blocks of very different sizes, zeros, and the type's extremes: each block keeps its own scale."""
    n, k = 64, 2048
    _, packed, w, mag = make(dev, wtype, n, k, 9)
    g = torch.Generator(device=dev).manual_seed(4)
    e = torch.randint(-60, 60, (2, k // 32, 1), generator=g, device=dev).float()
    x = (torch.randn(2, k // 32, 32, generator=g, device=dev) * torch.exp2(e)).view(2, k)
    x[:, 64:128] = 0
    x[0, 256:288] = 1e-42  # subnormal
    x[1, 300] = 1e30
    y = b2q.mul_vec(wtype, packed, n, k, x)
    assert bool(((y.double() - x.double() @ w.t()).abs() <= bound(x, mag, k) + 1e-44).all())
    z = b2q.mul_vec(wtype, packed, n, k, torch.zeros(3, k, device=dev))
    assert bool((z == 0).all())
    tiny = torch.full((1, k), 1e-42, device=dev)  # nothing but subnormals: the block scale's lowest value
    y = b2q.mul_vec(wtype, packed, n, k, tiny)
    assert bool((y.double() - tiny.double() @ w.t()).abs().max() <= k * 2.0 ** -149)


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
@pytest.mark.parametrize("v", [float("inf"), float("-inf"), float("nan")])
def test_nonfinite_activations_stay_in_their_token(dev, wtype, v):
    n, k = 100, 512
    _, packed, w, mag = make(dev, wtype, n, k, 2)
    x = torch.randn(3, k, device=dev)
    x[1, 77] = v
    y = b2q.mul_vec(wtype, packed, n, k, x)
    assert not bool(torch.isfinite(y[1]).any())
    ref = x[[0, 2]].double() @ w.t()
    assert bool(((y[[0, 2]].double() - ref).abs() <= bound(x[[0, 2]], mag, k)).all())


def test_matches_dequantize_and_strict_mul_mat(dev):
    """The same arithmetic contract as the fp32 path with the dequantized weight."""
    for wtype in (b2q.TYPE_Q4_0, b2q.TYPE_Q4_K):
        raw, packed, w, mag = make(dev, wtype, 300, 1024, 21)
        x = torch.randn(4, 1024, device=dev)
        strict = b2q.mul_mat_f32(b2q.dequantize(wtype, raw, 1024), x)
        y = b2q.mul_vec(wtype, packed, 300, 1024, x)
        # both within their bounds of the exact product: the strict path's chain has k roundings
        lim = bound(x, mag, 1024) + 1024 ** 0.5 * 2.0 ** -23 * (x.double().abs() @ mag.t())
        assert bool(((y - strict).double().abs() <= lim).all())


def test_repeats_bit_for_bit_and_empty(dev):
    _, packed, _, _ = make(dev, b2q.TYPE_Q4_K, 3000, 2048, 1)
    x = torch.randn(2, 2048, device=dev)
    y = b2q.mul_vec(b2q.TYPE_Q4_K, packed, 3000, 2048, x)
    for _ in range(3):
        assert torch.equal(b2q.mul_vec(b2q.TYPE_Q4_K, packed, 3000, 2048, x), y)
    assert b2q.mul_vec(b2q.TYPE_Q4_K, packed, 3000, 2048, x[:0]).shape == (0, 3000)


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
@pytest.mark.parametrize("n,k,m,xt", [
    (200, 4096, 1, "f16"), (41, 2048, 8, "bf16"), (1500, 4352, 4, "f32"), (1, 16384, 3, "f32"), (6000, 4096, 8, "f32"),
    (3001, 8448, 6, "bf16"), (1000, 16128, 2, "f32"), (2500, 11264, 5, "f16"), (12001, 4096, 7, "f32"),
])
def test_long_rows_shared_out(dev, wtype, n, k, m, xt):
    """Rows long beside their number: several CTAs share them out.  Bias, gate and the residual in place are added
    once, the result repeats bit for bit, and a captured call on another stream gives it too."""
    _, packed, w, mag = make(dev, wtype, n, k, n + k + 1)
    g = torch.Generator(device=dev).manual_seed(m)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, bias, gate, base = rand(m, k).to(DT[xt]), rand(n), rand(n), rand(m, n + 5)
    ref, tol = x.double() @ w.t(), bound(x, mag, k)
    r1 = ref + bias.double()
    r2 = base[:, :n].double() + gate.double() * r1
    lim = tol * gate.double().abs() + 2.0 ** -22 * ((gate.double() * r1).abs() + r2.abs())
    outs = []
    for _ in range(3):
        y = base.clone()
        b2q.mul_vec(wtype, packed, n, k, x, bias=bias, gate=gate, resid=y[:, :n], out=y[:, :n])
        outs.append(y)
    assert bool(((outs[0][:, :n].double() - r2).abs() <= lim).all())
    assert torch.equal(outs[0][:, n:], base[:, n:])
    assert torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])
    plain = b2q.mul_vec(wtype, packed, n, k, x)
    assert bool(((plain.double() - ref).abs() <= tol).all())
    side = torch.cuda.Stream()
    y = torch.zeros(m, n, device=dev)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b2q.mul_vec(wtype, packed, n, k, x, out=y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, plain)


# Activations that do not fit a CTA's shared memory (split into digits chunk by chunk, the sums kept in between), with
# one and with several row tiles a CTA; CTAs that own more row tiles than they keep sums of, with and without chunks; and
# the same for the CTAs of a cluster.
@pytest.mark.parametrize("wtype,n,k,m,xt", [
    (b2q.TYPE_Q4_0, 53, 65536, 3, "f32"), (b2q.TYPE_Q4_0, 53, 65536, 8, "f16"), (b2q.TYPE_Q4_0, 40, 65568, 5, "bf16"),
    (b2q.TYPE_Q4_0, 17, 131104, 8, "f32"), (b2q.TYPE_Q4_K, 53, 65536, 4, "f32"), (b2q.TYPE_Q4_K, 70, 65536, 8, "bf16"),
    (b2q.TYPE_Q4_K, 1, 22784, 8, "f32"), (b2q.TYPE_Q4_0, 20000, 6432, 8, "f32"), (b2q.TYPE_Q4_K, 20000, 6400, 7, "f16"),
    (b2q.TYPE_Q4_0, 79000, 3360, 8, "f32"), (b2q.TYPE_Q4_K, 78506, 3328, 8, "f32"),
    (b2q.TYPE_Q4_0, 38419, 1888, 7, "f32"), (b2q.TYPE_Q4_0, 38419, 1888, 8, "bf16"), (b2q.TYPE_Q4_K, 37927, 2048, 6, "f32"),
    (b2q.TYPE_Q4_K, 56881, 6400, 2, "bf16"), (b2q.TYPE_Q4_0, 56881, 5408, 4, "f32"),
])
def test_chunks_and_groups_of_tiles(dev, wtype, n, k, m, xt):
    rows = torch.arange(n, device=dev) % 1009  # (1009 rows over and over: quick to make)
    raw, _, w, mag = make(dev, wtype, min(n, 1009), k, n + k + 2)
    raw = raw[rows].contiguous()
    packed = b2q.weight_pack_q4_0(raw, k) if wtype == b2q.TYPE_Q4_0 else b2q.weight_pack(wtype, raw, k)
    g = torch.Generator(device=dev).manual_seed(m + 1)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, bias, gate, base = rand(m, k).to(DT[xt]), rand(n), rand(n), rand(m, n + 3)
    ref, tol = (x.double() @ w.t())[:, rows], bound(x, mag, k)[:, rows]
    plain = b2q.mul_vec(wtype, packed, n, k, x)
    assert bool(((plain.double() - ref).abs() <= tol).all())
    r1 = ref + bias.double()
    r2 = base[:, :n].double() + gate.double() * r1
    lim = tol * gate.double().abs() + 2.0 ** -22 * ((gate.double() * r1).abs() + r2.abs())
    y = base.clone()
    b2q.mul_vec(wtype, packed, n, k, x, bias=bias, gate=gate, resid=y[:, :n], out=y[:, :n])
    assert bool(((y[:, :n].double() - r2).abs() <= lim).all())
    assert torch.equal(y[:, n:], base[:, n:])
    assert torch.equal(b2q.mul_vec(wtype, packed, n, k, x), plain)
