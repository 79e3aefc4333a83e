"""Paged attention (b2q_attention_paged) where rows and keys are unusual: rows without a key beside rows with some,
values near the type's limits, infinities, scores far below a row's largest."""
import math

import pytest
import torch

import b2q
from test_gpu_attention_paged import DT, check, make, reference

pytestmark = pytest.mark.gpu


# 4 / 2 heads: two rows a token; up to 32 and 128 rows (rows kernel), more (tile kernel); announced lengths that give
# one stretch of the keys and several
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [3, 2, 20, 6], [150, 130, 40, 300], [70, 64, 65, 200]])
@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "bf16"), (64, "f16"), (128, "f16")])
@pytest.mark.parametrize("max_kv", [700, 20000])
def test_rows_without_keys_are_zero(dev, news, D, dt, max_kv):
    """No keys, fewer keys than new tokens (rows before the first key beside rows that see some), absent pages at the
    front, in the middle and everywhere: rows that see nothing are exactly 0."""
    lens = [0, max(1, news[1] // 2), 500, 700]
    q, kc, vc, table, L, cu = make(dev, lens, news, 4, 2, D, DT[dt], 32, seed=7)
    table[2] = -1
    table[3, 2:5] = -1
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max_kv, 4)
    ref, mag = reference(q, kc, vc, table, L, cu, 4)
    check(o, ref, mag, DT[dt])
    blind = mag.sum(1) == 0
    assert int(blind.sum()) >= news[0] + news[2] + news[1] - lens[1]
    assert bool((o[blind] == 0).all())


@pytest.mark.parametrize("D,dt", [(64, "bf16"), (128, "bf16"), (128, "f16")])
@pytest.mark.parametrize("max_kv", [700, 20000])
def test_window_without_pages(dev, D, dt, max_kv):
    """A window whose pages are absent for some rows of a chunk and present for others."""
    q, kc, vc, table, L, cu = make(dev, [700, 460], [300, 200], 4, 2, D, DT[dt], 32, seed=8)
    table[0, 12:17] = -1   # keys 384 to 543: rows at 450 to 543 with a window of 64 see none
    table[1, 10:] = -1
    o = b2q.attention_paged(q, kc, vc, table, L, cu, 300, max_kv, 4, window=64)
    ref, mag = reference(q, kc, vc, table, L, cu, 4, window=64)
    check(o, ref, mag, DT[dt])
    blind = mag.sum(1) == 0
    assert int(blind.sum()) > 100 and bool((o[blind] == 0).all())


@pytest.mark.parametrize("news,lens", [([5, 3], [300, 64]), ([200, 131], [500, 131]), ([300, 40], [3000, 900])])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("max_kv", [None, 20000])
def test_huge_values_of_unseen_keys(dev, news, lens, D, max_kv):
    """Finite bf16 values of 1e36 in later tokens' keys do not reach the rows before them (2^-125 of them would)."""
    q, kc, vc, table, L, cu = make(dev, lens, news, 4, 2, D, torch.bfloat16, 32, seed=9)
    for b in range(2):
        for key in (lens[b] - 1, lens[b] - news[b] // 2):
            vc[int(table[b, key // 32]), :, key % 32] = 1e36
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens) if max_kv is None else max_kv, 4)
    ref, mag = reference(q, kc, vc, table, L, cu, 4)
    check(o, ref, mag, torch.bfloat16)


@pytest.mark.parametrize("news,lens", [([1, 1], [400, 77]), ([70, 150], [400, 150])])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_infinite_scores_under_a_negative_scale(dev, news, lens, D, dt):
    """A product of -infinity is a score of +infinity when the scale is negative, and rows that see it are NaN."""
    q, kc, vc, table, L, cu = make(dev, lens, news, 4, 2, D, DT[dt], 16, seed=2)
    q.abs_().add_(0.25)  # (no zeros: they would give NaN themselves)
    kc[int(table[0, 1]), :, 3, 9] = -math.inf
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), 4, scale=-0.1)
    assert bool(torch.isnan(o[:int(cu[1])]).all())
    ref, mag = reference(q, kc, vc, table, L, cu, 4, scale=-0.1)
    check(o[int(cu[1]):], ref[int(cu[1]):], mag[int(cu[1]):], DT[dt])


def same_kind(got, ref):
    """NaN, +infinity and -infinity in the same places."""
    return all(torch.equal(f(got), f(ref)) for f in (torch.isnan, torch.isposinf, torch.isneginf))


# rows kernel (one stretch, a cluster, stretches joined afterwards; 16 and 32 rows), tile kernel (whole and split)
@pytest.mark.parametrize("Hq,news,lens,max_kv", [
    (4, [1, 1], [100, 33], None), (4, [1, 1], [900, 333], None), (4, [1, 1], [9000, 333], None), (24, [2, 1], [100, 40], None),
    (24, [2, 1], [5000, 40], None), (4, [150, 140], [400, 140], None), (4, [150, 140], [400, 140], 20000),
])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16"), (128, "f16"), (64, "bf16")])
@pytest.mark.parametrize("scale", [0.125, 0.4])
def test_infinite_values_reach_rows_that_see_them(dev, Hq, news, lens, max_kv, D, dt, scale):
    """An infinite value of a key that a row sees makes that output the infinity, however small the key's weight;
    infinities of both signs, or a NaN, make it NaN.  Weights stay above 2^-126 of a row's largest."""
    q, kc, vc, table, L, cu = make(dev, lens, news, Hq, 2, D, DT[dt], 16, seed=Hq + D)
    q *= 0.5
    at = lambda b, key: (int(table[b, key // 16]), slice(None), key % 16)  # noqa: E731
    for b in range(2):
        vc[at(b, 3)][:, 5] = math.inf
        vc[at(b, lens[b] // 2)][:, 6] = -math.inf
        vc[at(b, 1)][:, 7] = math.inf
        vc[at(b, lens[b] // 3)][:, 7] = -math.inf
        vc[at(b, 2)][:, 8] = math.nan
        vc[at(b, lens[b] - 1)][:, 9] = math.inf
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens) if max_kv is None else max_kv, Hq, scale=scale)
    ref, mag = reference(q, kc, vc, table, L, cu, Hq, scale=scale)
    assert bool(torch.isposinf(ref).any()) and bool(torch.isneginf(ref).any()) and bool(torch.isnan(ref).any())
    assert same_kind(o, ref.to(DT[dt]))
    fin = torch.isfinite(ref)
    check(torch.where(fin, o, 0), torch.where(fin, ref, 0.0), torch.where(fin, mag, 0.0), DT[dt])


@pytest.mark.parametrize("Hq,news,lens", [(4, [1], [700]), (24, [2], [5000]), (4, [150], [400])])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_infinite_value_of_a_light_key(dev, Hq, news, lens, dt):
    """The key with the infinity weighs 2^-60 of the others: still the infinity."""
    D = 64
    q, kc, vc, table, L, cu = make(dev, lens, news, Hq, 2, D, DT[dt], 16, seed=3)
    q.fill_(1.0)
    kc.zero_()
    pg, off = int(table[0, 1]), 4
    kc[pg, :, off] = -5.25     # 64 * 5.25 / 8 = 42 below the others: 2^-60.6
    vc[pg, :, off, 11] = -math.inf
    o = b2q.attention_paged(q, kc, vc, table, L, cu, max(news), max(lens), Hq)
    ref, _ = reference(q, kc, vc, table, L, cu, Hq)
    assert bool(torch.isneginf(ref).any()) and same_kind(o, ref.to(DT[dt]))
