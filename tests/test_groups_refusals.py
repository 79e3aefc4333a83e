"""Refusals of the calls for rows that go by group, and what their wrappers pass on, beyond test_groups_abi.py and
test_groups_wrappers.py; no GPU needed."""
import pytest
import torch

import b2q
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
