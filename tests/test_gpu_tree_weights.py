"""Weights of the attention of drafted trees keep 16 bits in every form of the kernel, so that a row does not lose digits because others share its call.

The bound per element.  The result's one rounding: 2^-8 |o|.  A weight enters the product as two bf16 pieces, the second one the first's remainder: each rounding
leaves 2^-8 of what it rounds, so 2^-16 of the weight is lost.  Scores are off by (dim + 8) 2^-23 scale sum |q k|, which a weight sees twice (itself and the sum);
the exponential and the fp32 sums of up to 2^11 weights take 2^-22 + (2^11 / 32 + 16) 2^-23 (32 sums run beside each other), below 2^-16; the tensor core adds 16
products at a time to a running sum that it does not round to nearest, 2 (2^11 / 16) times: 2^8 2^-23 = 2^-15.  All in units of sum p |v|."""

import pytest
import torch

from glm_tpu_b200.layers.attention import paged

from tests.paged_cases import to_cuda, tree_case, tree_exact


def tight(case):
    """``(result, bound)``: ``tree_exact``'s bound holds 2^-8 for the weights; that is taken out and the terms above put in."""
    want, loose = tree_exact(case)
    c = case["cache"]
    weighed = tree_exact(case | {"cache": paged.PagedKV(c.k, c.v.abs(), c.table)})[0]  # sum p |v|
    return want, loose + (2.0**-16 + 2.0**-16 + 2.0**-15 - 2.0**-8) * weighed


@pytest.mark.gpu
@pytest.mark.parametrize("lengths, sizes, H, G, dim, page", [
    ([1900], [64], 8, 1, 128, 64), ([700, 5, 1000], [40, 3, 17], 16, 2, 64, 16), ([1200], [60], 64, 8, 128, 128), ([333, 1500], [64, 64], 4, 1, 80, 48),  # two tiles a unit
    ([1900], [16], 8, 1, 128, 64), ([900, 40], [5, 2], 16, 4, 64, 16), ([1500], [9], 6, 3, 192, 8), ([300, 400], [8, 8], 8, 2, 128, 64)])
def test_weights_keep_their_digits(native_lib, lengths, sizes, H, G, dim, page):
    case = tree_case(lengths, sizes, H=H, G=G, dim=dim, vdim=dim, page=page, seed=3)
    off = (paged.tree_attention(**to_cuda(case)).cpu().double() - tight(case)[0]).abs()
    bound = tight(case)[1]
    assert bool((off <= bound).all()), (float((off - bound).max()), int((off > bound).sum()))
