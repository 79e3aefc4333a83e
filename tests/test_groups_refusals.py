"""Refusals of the calls for rows that go by group, and what their wrappers pass on, beyond test_groups_abi.py and
test_groups_wrappers.py; no GPU needed."""
import pytest
import torch

import b2q
import cached_block as cb
import test_groups_abi as abi
from test_groups_wrappers import lib_calls, refused, route, z  # noqa: F401


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
