"""Refusals of the calls for rows that go by group, and what their wrappers pass on, beyond test_groups_abi.py and
test_groups_wrappers.py; no GPU needed."""
import pytest
import torch

import b2q
import cached_block as cb
import test_groups_abi as abi
from test_groups_wrappers import F16, F32, I32, join, lib_calls, lora, mmid, refused, route, verify, z  # noqa: F401


@pytest.mark.parametrize("sc", [2, 3, 6, 8, -1, -4])
def test_route_scorings_that_do_not_exist(b2q_mod, sc):
    assert abi.route(sc=sc) == abi.ARG


def test_route_passes_where_the_bias_goes(lib_calls):
    route(bias=z(8), scoring="sigmoid")
    route(bias=z(8), scoring="sigmoid", bias_on="score")
    route(bias=z(8), bias_on="score")
    assert [c[1][7] for c in lib_calls] == [1, 5, 4]
    lib_calls.clear()
    refused(lib_calls, route, bias_on="weights")


@pytest.mark.parametrize("names", [("fc1",), ("fc2",), ("qkv", "out", "fc2"), ("fc1", "fc2")])
def test_a_block_with_experts_refuses_adapters_of_the_linears_it_does_not_have(names):
    block = cb.CachedBlock.__new__(cb.CachedBlock)
    block.experts = object()
    adapters = cb.Adapters({n: (z(2, 8, 32, dt=torch.float16), z(2, 32, 8, dt=torch.float16)) for n in names})
    with pytest.raises(ValueError):
        block.forward(z(3, 32), None, 0, {}, None, adapters=adapters, rows=(None, None))


@pytest.mark.parametrize("pairs", [{}, {"gate": (z(2, 8, 32), z(2, 32, 8))}, {"qkv": (z(2, 8, 32), z(2, 32, 8)), "o": None}])
def test_adapters_of_unknown_linears_are_refused(pairs):
    with pytest.raises(ValueError):
        cb.Adapters(pairs)


@pytest.mark.parametrize("scales", [z(5), z(6, dt=F16), z(12)[::2]])
def test_lora_refuses_row_scales(lib_calls, scales):
    refused(lib_calls, lora, row_scales=scales)


def test_lora_passes_row_scales(lib_calls):
    b2q._lib.b2q_lora_add_rows = lambda *a: (lib_calls.append(("rows", a)), 0)[1]
    s = z(6)
    lora(row_scales=s)
    assert [c[0] for c in lib_calls] == ["rows"] and lib_calls[0][1][11] == s.data_ptr() and len(lib_calls[0][1]) == 22


def lora_rows(rs, **kw):
    a = dict(xt=1, x=abi.FAKE, T=8, k=64, ldx=128, a=abi.FAKE, b=abi.FAKE, G=3, r=16, n=32, sc=abi.FAKE, order=abi.FAKE, off=abi.FAKE,
             yt=0, res=abi.FAKE, ldr=128, y=abi.FAKE, ldy=128, ws=abi.FAKE, wsb=abi.BIG)
    a.update(kw)
    return b2q.lib().b2q_lora_add_rows(a["xt"], a["x"], a["T"], a["k"], a["ldx"], a["a"], a["b"], a["G"], a["r"], a["n"], a["sc"], rs,
                                       a["order"], a["off"], a["yt"], a["res"], a["ldr"], a["y"], a["ldy"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("rs,kw,expect", [(abi.FAKE + 2, {}, abi.ALIGN), (abi.FAKE, dict(r=12), abi.ARG), (None, dict(T=0), abi.OK),
                                          (abi.FAKE, dict(T=0), abi.OK), (abi.FAKE, dict(T=5000, ws=None), abi.WS)])
def test_lora_rows_checks(b2q_mod, rs, kw, expect):
    assert lora_rows(rs, **kw) == expect


# ------------------------------------------------------------------ results on operands, and on one another
# Buffers a megabyte apart, so that only what a case moves lies on something.
MB = 1 << 20


def at(i):
    return 64 * MB + i * MB


def apart_route(**kw):
    a = dict(x=at(0), bias=at(1), ids=at(2), w=at(3), order=at(4), off=at(5), ws=at(6), T=400, top=2)
    a.update(kw)
    return abi.route(**a)


def apart_rows(**kw):
    a = dict(ids=at(0), order=at(1), off=at(2), ws=at(3), S=3000)
    a.update(kw)
    return abi.rows(**a)


def apart_mmid(**kw):
    a = dict(w=at(0), x=at(1), order=at(2), off=at(3), bias=at(4), y=at(5))
    a.update(kw)
    return abi.mmid(**a)


def apart_join(**kw):
    a = dict(y=at(0), w=at(1), ids=at(2), r=at(3), o=at(4))
    a.update(kw)
    return abi.join(**a)


def apart_lora(**kw):
    a = dict(x=at(0), a=at(2), b=at(3), sc=at(4), order=at(5), off=at(6), res=at(8), y=at(10), ws=at(12), T=2000)
    a.update(kw)
    return lora_rows(at(7), **a)


def apart_verify(**kw):
    a = dict(t=at(0), g=at(1), d=at(2), cu=at(3), u=at(4), v=at(5), acc=at(6), tok=at(7))
    a.update(kw)
    return abi.verify(**a)


CALLS = [
    (apart_route, [("ids", [at(0), at(0) + 32 * 400 - 4, at(1) + 28, at(1) - 3196, at(3), at(4), at(5), at(6)]), ("w", [at(0), at(1), at(4)]),
                   ("order", [at(0) + 32, at(1), at(5) - 3196]), ("off", [at(0), at(1) - 32]), ("ws", [at(0), at(1), at(2) + 3196])]),
    (apart_rows, [("order", [at(0), at(0) + 11996, at(2), at(3)]), ("off", [at(0) + 4, at(3)]), ("ws", [at(0)])]),
    (apart_mmid, [("y", [at(0), at(0) + 3 * 2048 + 15 * 128 + 96, at(1), at(2) + 76, at(3) + 16, at(4) + 252, at(4) - 32 * 19 - 30])]),
    (apart_join, [("o", [at(0), at(1) + 28, at(2) - 64 * 3 - 60, at(2), at(3) + 64])]),
    (apart_lora, [("y", [at(0), at(2) + 3 * 16 * 64 * 2 - 4, at(3), at(4) + 8, at(5), at(6) + 12, at(7) + 7996, at(8) + 128, at(12)]),
                  ("ws", [at(0), at(2), at(3), at(4), at(5), at(6), at(7), at(8), at(10)])]),
    (apart_verify, [("acc", [at(0), at(1), at(2), at(3) + 12, at(4), at(5), at(7) + 32]),
                    ("tok", [at(0) + 400 * 8 + 396, at(1), at(2) + 20, at(3), at(4) - 32, at(5)])]),
]


@pytest.mark.parametrize("call,name,where", [(c, n, p) for c, moves in CALLS for n, ps in moves for p in ps])
def test_results_on_any_operand_are_refused(b2q_mod, call, name, where):
    assert call(**{name: where}) == abi.ARG


def one_row(width, step, dt):
    """A row of a table whose rows are `step` values apart."""
    return z(3, step, dt=dt)[1:2, :width]


def test_the_stride_of_a_single_row_does_not_matter(lib_calls):
    """Rows cut out of tables of any width, and results that are the residual by another view of it."""
    mmid(rows=1, per_row=1, x=one_row(64, 99, F16), order=z(1, dt=I32), out=one_row(16, 33, F16))
    resid = one_row(16, 50, F32)
    join(T=1, y=one_row(16, 77, F16), weights=z(1, 1), ids=z(1, 1, dt=I32), resid=resid, out=resid.view(16).unsqueeze(0))
    join(T=1, y=one_row(16, 77, F16), weights=z(1, 1), ids=z(1, 1, dt=I32), out=one_row(16, 5000, F32))
    lora(T=1, x=one_row(64, 67, F16), resid=one_row(32, 41, F32), order=z(1, dt=I32))
    route(T=1, logits=one_row(8, 13, F32))
    verify(B=1, D=0, target=one_row(20, 23, F32), draft_probs=z(0, 20), drafts=z(0, dt=I32), u=z(0), v=z(1))
    a = [c[1] for c in lib_calls]
    assert a[0][9] == 128 and a[0][18] == 32
    assert a[1][2] == 32 and a[1][10] == a[1][12] == 64 and a[1][9] == a[1][11]
    assert a[2][2] == 32 and a[2][12] == 64
    assert a[3][4] == 128 and a[3][15] == a[3][17] == 128
    assert a[4][4] == 32 and a[5][2] == 80


def test_strides_of_more_rows_are_passed(lib_calls):
    join(y=z(8, 20, dt=F16)[:, :16], out=z(4, 40)[:, :16])
    lora(x=z(6, 72, dt=F16)[:, :64], resid=z(6, 40)[:, :32])
    route(logits=z(5, 11)[:, :8])
    verify(target=z(8, 24)[:, :20], draft_probs=z(5, 28)[:, :20])
    a = [c[1] for c in lib_calls]
    assert a[0][2] == 40 and a[0][12] == 160 and a[1][4] == 144 and a[1][15] == 160 and a[2][4] == 44 and a[3][2] == 96 and a[3][4] == 112


def test_workspaces_of_plans(b2q_mod):
    """None for one launch; the counts of every run for two."""
    L = b2q.lib()
    for T, E, top, need in [(0, 64, 4, 0), (64, 64, 4, 0), (65, 64, 4, 3 * 65 * 4), (32, 65, 4, 0), (33, 65, 4, 2 * 66 * 4),
                            (33, 64, 5, 2 * 65 * 4), (4736, 64, 1, 148 * 65 * 4), (100000, 1024, 1, 148 * 1025 * 4)]:
        assert L.b2q_moe_route_workspace_bytes(T, E, top) == need
    for S, G, need in [(0, 8, 0), (2048, 8, 0), (2049, 8, 5 * 9 * 4), (1000000, 1024, 148 * 1025 * 4)]:
        assert L.b2q_group_rows_workspace_bytes(S, G) == need
