"""b2q_draft_verify against the definition in 64 bits; the results are whole numbers and have to be equal."""
import math

import numpy as np
import pytest
import torch

import b2q

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def reference(target, guess, drafts, cu, u, v):
    clean = lambda p: np.where(np.isfinite(p) & (p > 0), p, 0.0)  # noqa: E731
    target = target.double().cpu().numpy()
    guess = None if guess is None else guess.double().cpu().numpy()
    drafts, cu, u, v = (t.cpu().numpy() for t in (drafts, cu, u, v))
    V = target.shape[1]
    accepted, out = [], []
    for b in range(len(cu) - 1):
        new, weight = [], None
        for i in range(cu[b], cu[b + 1]):
            p, d = target[i + b], drafts[i]
            q = np.zeros(V) if guess is None else guess[i]
            if guess is None and 0 <= d < V:
                q[d] = 1.0
            with np.errstate(invalid="ignore"):
                if 0 <= d < V and float(u[i]) * q[d] < p[d]:
                    new.append(int(d))
                    continue
                weight = np.where((p > q) & np.isfinite(p) & (p > 0), p - np.maximum(q, 0.0), 0.0)
            if weight.sum() == 0:
                weight = clean(p)
            break
        if weight is None:
            weight = clean(target[cu[b + 1] + b])
        edge = np.cumsum(weight)
        if edge[-1] > 0:
            vb = float(v[b])
            j = int(np.searchsorted(edge, (vb if vb > 0 else 0.0) * edge[-1], side="right"))
            token = min(j, int(np.flatnonzero(weight).max()))
        else:
            token = -1
        accepted.append(len(new))
        out += new + [token] + [-1] * (cu[b + 1] - cu[b] - len(new))
    return accepted, out


def make(dev, counts, V, ty, seed=0, sharp=2.5, noise=0.7):
    g = torch.Generator(device=dev).manual_seed(seed)
    B, D = len(counts), sum(counts)
    logits = sharp * torch.randn(D + B, V, generator=g, device=dev)
    owner = torch.repeat_interleave(torch.arange(B, device=dev), torch.tensor(counts, device=dev))
    at = torch.arange(D, device=dev) + owner
    guess = torch.softmax(logits[at] + noise * torch.randn(D, V, generator=g, device=dev), -1)
    race = -torch.log(torch.rand(D, V, generator=g, device=dev).clamp(min=1e-30))
    drafts = (guess / race).argmax(-1).int() if D else torch.zeros(0, dtype=torch.int32, device=dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=dev)
    return [torch.softmax(logits, -1).to(DT[ty]), guess.to(DT[ty]), drafts, cu, torch.rand(D, generator=g, device=dev),
            torch.rand(B, generator=g, device=dev)]


def check(args):
    accepted, tokens = b2q.draft_verify(*args)
    ra, rt = reference(*args)
    assert accepted.tolist() == ra
    assert tokens.tolist() == rt


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("counts,V", [([1], 1), ([0], 5), ([3, 0, 2], 2), ([2, 5, 1], 33), ([4] * 20, 1000),
                                      ([1, 2, 3, 4], 32000), ([7, 0, 3] * 5, 50257), ([40, 33, 70], 600), ([2, 3], 151001)])
def test_draft_verify(dev, ty, counts, V):
    args = make(dev, counts, V, ty, seed=V)
    check(args)
    check([args[0], None] + args[2:])


def test_kept_shares_and_draws_follow_the_target(dev):
    """The first token of many requests with one draft is distributed as the target, whatever the draft model."""
    B, V = 20000, 6
    g = torch.Generator(device=dev).manual_seed(3)
    p = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.2, 0.1], device=dev)
    q = torch.tensor([0.1, 0.4, 0.1, 0.2, 0.1, 0.1], device=dev)
    drafts = torch.multinomial(q, B, replacement=True, generator=g).int()
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    u, v = torch.rand(B, generator=g, device=dev), torch.rand(B, generator=g, device=dev)
    _, tokens = b2q.draft_verify(p.repeat(2 * B, 1), q.repeat(B, 1), drafts, cu, u, v)
    share = torch.bincount(tokens[0::2].long(), minlength=V).double() / B
    # five standard deviations of a share of B draws
    assert bool(((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt()).all())


def test_borders(dev):
    """Numbers at the ends: v 0 and just below 1, past 1, negative, NaN; u 0 and 1; zeros at the row's ends."""
    V = 900
    p = torch.zeros(12, V, device=dev)
    p[:, 5:700] = torch.rand(12, 695, device=dev)
    p[:, 300:600] = 0
    cu = torch.zeros(13, dtype=torch.int32, device=dev)
    v = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 1e-30, 0.5, 0.25, 0.75, 0.999999, math.inf], device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    accepted, tokens = b2q.draft_verify(p, None, none, cu, torch.zeros(0, device=dev), v)
    assert accepted.tolist() == [0] * 12
    got, want = tokens.tolist(), reference(p, None, none, cu, torch.zeros(0), torch.nan_to_num(v, nan=0.0, posinf=2.0))[1]
    assert got == want
    assert got[0] == 5 and got[2] == got[3] == got[11] == 699 and got[4] == got[5] == 5


def test_equal_models_keep_every_draft(dev):
    args = make(dev, [5] * 30, 3000, "f32", seed=2, noise=0.0)
    accepted, tokens = b2q.draft_verify(*args)
    assert accepted.tolist() == [5] * 30
    check(args)


def test_nothing_above_the_draft(dev):
    """A draft that is turned down although the target is nowhere above the draft model: the draw is the target's."""
    V = 500
    p = torch.full((2, V), 1.0 / V, device=dev)
    q = torch.full((1, V), 2.0 / V, device=dev)
    args = [p, q, torch.tensor([7], dtype=torch.int32, device=dev), torch.tensor([0, 1], dtype=torch.int32, device=dev),
            torch.tensor([0.9], device=dev), torch.tensor([0.5], device=dev)]
    check(args)
    assert b2q.draft_verify(*args)[0].tolist() == [0]


def test_rows_with_nothing_and_with_no_numbers(dev):
    args = make(dev, [2, 2, 2, 1], 700, "f32", seed=6)
    args[0][0] = 0.0
    args[0][3] = math.nan
    args[0][6, ::2] = math.nan
    args[0][6, 1] = math.inf
    args[1][5, ::3] = math.nan
    args[1][5, 1::3] = -0.5
    args[0][9] = -1.0
    check(args)


def test_drafts_outside_the_vocabulary_are_turned_down(dev):
    args = make(dev, [3, 2, 4], 100, "f32", seed=8)
    args[2][0], args[2][3], args[2][6] = -1, 100, 1 << 30
    args[4].zero_()
    check(args)
    check([args[0], None] + args[2:])


def test_row_strides(dev):
    args = make(dev, [2, 3, 1], 333, "f16", seed=9)
    for i in (0, 1):
        wide = torch.full((args[i].shape[0], 400), 0.5, dtype=torch.float16, device=dev)
        wide[:, 7:340] = args[i]
        args[i] = wide[:, 7:340]
    check(args)


def test_no_requests(dev):
    z = torch.zeros(0, device=dev)
    i = torch.zeros(1, dtype=torch.int32, device=dev)
    accepted, tokens = b2q.draft_verify(torch.zeros(0, 10, device=dev), None, i[:0], i, z, z)
    assert accepted.numel() == 0 and tokens.numel() == 0


def test_broken_offsets_stay_inside(dev):
    args = make(dev, [3, 2, 4], 100, "f32", seed=8)
    args[3] = torch.tensor([-4, 1 << 30, 2, 5], dtype=torch.int32, device=dev)
    b2q.draft_verify(*args)
    torch.cuda.synchronize()


def test_in_a_graph(dev):
    args = make(dev, [3, 0, 6, 2], 5000, "bf16", seed=1)
    b2q.draft_verify(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accepted, tokens = b2q.draft_verify(*args)
    for seed in (2, 3):
        for t, new in zip(args, make(dev, [3, 0, 6, 2], 5000, "bf16", seed=seed)):
            t.copy_(new)
        graph.replay()
        ra, rt = reference(*args)
        assert accepted.tolist() == ra and tokens.tolist() == rt


def test_rows_behind_the_last_request_are_empty(dev):
    """A batch with room for more drafts than it has: the tokens behind its last request are -1, its others as ever."""
    args = make(dev, [3, 1, 2, 4], 200, "f32", seed=5)
    args[3] = torch.tensor([0, 3, 4, 6], dtype=torch.int32, device=dev)  # three requests of 6 drafts; 10 are there
    args[0], args[5] = args[0][:13], args[5][:3]
    accepted, tokens = b2q.draft_verify(*args)
    ra, rt = reference(args[0], args[1], args[2], args[3], args[4], args[5])
    assert accepted.tolist() == ra and tokens.tolist() == rt + [-1] * 4
