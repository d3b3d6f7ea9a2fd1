"""Groups scored by the sum of their two largest members (b200dnn_moe_gate) where a bias makes the two large and of opposite sign: their sum is small, its rounding errors are the members'."""
import numpy as np
import pytest
import torch

from test_moe_gate_gpu import capi, check, logits  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [3.0, 1000.0, 1e6])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,k,groups,top_groups", [(8, 1, 4, 1), (64, 4, 32, 5), (64, 6, 32, 31), (16, 2, 8, 3)])
def test_members_that_cancel(capi, E, k, groups, top_groups, score, size):  # noqa: F811
    """Groups of two with biases of plus and minus one size: the groups' order is that of sums of scores, which one part in 2^24 of the size hides."""
    rng = np.random.default_rng(E)
    bias = np.where(np.arange(E) % 2 == 0, size, -size).astype(np.float32)
    check(capi, logits(400, E, seed=7), k, bias, score, groups, top_groups, "top2", False, 1.0)
    check(capi, logits(400, E, seed=8, spread=0.01), k, bias[rng.permutation(E // 2).repeat(2) * 2 + np.tile([0, 1], E // 2)], score, groups, top_groups, "top2", False, 1.0)


@pytest.mark.parametrize("E,k,groups,top_groups", [(64, 4, 8, 4), (64, 4, 16, 3), (256, 8, 8, 4)])
def test_groups_that_a_bias_takes_out(capi, E, k, groups, top_groups):  # noqa: F811
    """Whole groups, and parts of groups, at minus infinity beside ordinary biases."""
    bias = (np.random.default_rng(1).standard_normal(E) * 0.1).astype(np.float32)
    bias[:E // groups] = -np.inf
    bias[2 * E // groups + 1:3 * E // groups] = -np.inf
    for score in ("sigmoid", "softmax"):
        check(capi, logits(500, E, seed=3), k, bias, score, groups, top_groups, "top2", True, 1.0)
