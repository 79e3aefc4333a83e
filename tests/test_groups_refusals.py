"""Refusals of the calls for rows that go by group, and what their wrappers pass on, beyond test_groups_abi.py and
test_groups_wrappers.py; no GPU needed."""
import pytest
import torch

import b2q
import cached_block as cb
import test_groups_abi as abi
from test_groups_wrappers import F16, lib_calls, lora, refused, route, z  # noqa: F401


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
