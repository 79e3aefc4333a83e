"""Calls for rows that go by group at the borders between their kernels' forms, against plain 64-bit arithmetic
(tolerances as in test_gpu_groups.py, and equality where every value is exact)."""
import numpy as np
import pytest
import torch

import b2q
from test_gpu_groups import call_experts, check_rows, experts_reference, make_experts

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
