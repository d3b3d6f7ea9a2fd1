"""The order of b200dnn_moe_gate where a bias makes scores of very different size neighbours: an expert that lies behind the last choice in 32 bits may have a score, and so an error,
many orders of magnitude above those of the experts in front of it.  Against the definition in 64 bits, as test_moe_gate_gpu.py."""
import numpy as np
import pytest
import torch

from test_moe_gate_gpu import capi, check  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def steps(rng, x, most):
    """x moved by up to `most` neighbouring floats."""
    x = x.astype(np.float32)
    for _ in range(most):
        x = np.where(rng.random(x.shape) < 0.5, np.nextafter(x, np.float32(np.inf)), x).astype(np.float32)
    return x


def cancelled(T, E, big, score, seed):
    """Tiny scores with no bias, or one of their own size, and `big` experts at random places whose bias is minus their score rounded to f32."""
    rng = np.random.default_rng(seed)
    x = rng.uniform(-22, -19, (T, E)).astype(np.float32)
    bias = np.where(rng.random(E) < 0.5, 0.0, rng.uniform(-2e-9, 2e-9, E)).astype(np.float32)
    at = rng.choice(E, big, replace=False)
    top = rng.uniform(0.5, 4.0, big).astype(np.float32)
    if score == "softmax":
        top -= top.max()
    x[:, at] = steps(rng, np.broadcast_to(top, (T, big)), 3)
    row = np.median(x, 0).astype(np.float64)
    row[at] = top
    s = 1.0 / (1.0 + np.exp(-row)) if score == "sigmoid" else np.exp(row - row.max()) / np.exp(row - row.max()).sum()
    bias[at] = -s[at].astype(np.float32)
    return torch.from_numpy(x), bias


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,big,k,groups,top_groups,group_score", [
    (3, 1, 1, 1, 1, "max"), (8, 2, 1, 1, 1, "max"), (8, 2, 3, 1, 1, "max"), (64, 6, 6, 1, 1, "max"), (64, 20, 8, 8, 4, "top2"), (60, 9, 4, 6, 3, "max"), (256, 32, 8, 8, 4, "top2"),
    (256, 3, 16, 1, 1, "max"), (1024, 40, 12, 1, 1, "max")])
def test_a_bias_that_undoes_a_large_score(capi, score, E, big, k, groups, top_groups, group_score):  # noqa: F811
    for seed in range(4):
        x, bias = cancelled(400, E, big, score, 10 * E + seed)
        check(capi, x, k, bias, score, groups, top_groups, group_score, False, 1.0)


def test_one_cancelled_score_beside_two_tiny_ones(capi):  # noqa: F811
    """Top 1 of three: the tiny two are far enough apart by their own errors, and the third is in front of them by less than the error of a score near one."""
    rng = np.random.default_rng(0)
    top = rng.uniform(0.5, 6.0, 250).astype(np.float32)
    for value in top[:40]:
        s = 1.0 / (1.0 + np.exp(-np.float64(value)))
        x = np.tile(np.array([-20.0, -21.0, value], np.float32), (7, 1))
        x[:, 2] = steps(rng, x[:, 2], 4)
        check(capi, torch.from_numpy(x), 1, np.array([0.0, 0.0, -np.float32(s)], np.float32), "sigmoid", 1, 1, "max", False, 1.0)
