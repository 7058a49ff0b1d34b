"""A committed value that is not finite: where it shows, and where it must not."""

import math

import pytest
import torch

from glm_tpu_b200.layers.attention import paged

from tests.paged_cases import to_cuda, tree_case, tree_exact


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim, H, tree", [(64, 8, 4), (64, 8, 12), (128, 8, 40), (256, 8, 3), (128, 2, 1)])
@pytest.mark.parametrize("length", [90, 700])
def test_a_committed_value_that_is_not_finite(native_lib, length, dim, H, tree, value):
    case = tree_case([length, 33], [tree, 3], H=H, G=2, dim=dim, vdim=dim, page=32, seed=4)
    c = case["cache"]
    v = c.v.clone()
    v[c.table[0, 50 // 32], 50 % 32, 1, 5] = value  # channel 5 of the second key head
    got = paged.tree_attention(**to_cuda(case | {"cache": paged.PagedKV(c.k, v, c.table)})).cpu().double()
    want, bound = tree_exact(case)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:tree, H // 2 :, 5] = True
    assert not bool(torch.isfinite(got[hit]).any())
    assert bool(((got - want).abs() <= bound)[~hit].all())
