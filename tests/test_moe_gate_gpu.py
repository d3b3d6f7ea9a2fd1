"""GPU tests of b200dnn_moe_gate against the definition in 64 bits: ids, counts and rows are equal; a weight is a score in f32 (an exponential, a sum and a quotient:
a few half steps) over a sum of such, times scale: 2^-19 relative, and 2^-22 of the scale where a score is nearly zero beside the rest (bf16-sized exponents far below the row's maximum)."""
import ctypes as C

import numpy as np
import pytest
import torch

from serving import gate, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


def check(capi, x, k, bias, score, groups, top_groups, group_score, renorm, scale, pad=0):
    T, E = x.shape
    wide = torch.full((T, E + pad), 1e30, dtype=x.dtype, device="cuda")
    wide[:, :E] = x.cuda()
    ids, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
    counts, rows = torch.full((E,), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    kw = dict(bias=None if bias is None else torch.from_numpy(bias).cuda(), score=score, num_groups=groups, topk_groups=top_groups, group_score=group_score, renorm=renorm, scale=scale)
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, capi.make_moe_gate(wide[:, :E], k, ids, w, expert_counts=counts, slot_to_row=rows, **kw)))
    want = gate(x.double().numpy(), k, score, bias, groups, top_groups, group_score, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), want[0])
    np.testing.assert_allclose(w.cpu().numpy(), want[1], rtol=2.0 ** -19, atol=1e-37)
    assert np.array_equal(counts.cpu().numpy(), want[2])
    assert np.array_equal(rows.cpu().numpy(), want[3])
    again = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, capi.make_moe_gate(wide[:, :E], k, again, **kw)))
    assert torch.equal(ids, again)


def logits(T, E, dt="f32", seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed + T * 1000 + E)
    return (torch.randn(T, E, generator=g) * spread).to(torch.float32 if dt == "f32" else torch.bfloat16)


@pytest.mark.parametrize("T", [1, 33, 700])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,top_groups,group_score", [
    (4, 2, 1, 1, "max"), (64, 6, 1, 1, "max"), (256, 8, 8, 4, "top2"), (60, 4, 6, 3, "max"), (1, 1, 1, 1, "max"), (33, 16, 1, 1, "max"), (160, 6, 8, 3, "max"), (130, 5, 10, 2, "top2"),
    (1000, 10, 1, 1, "max"), (1024, 16, 32, 4, "top2"), (32, 2, 32, 2, "top2"), (32, 3, 32, 3, "max"), (300, 7, 4, 4, "top2"), (512, 12, 16, 1, "max"), (16, 16, 4, 4, "top2"), (96, 9, 3, 2, "top2")])
def test_forms(capi, T, dt, score, E, k, groups, top_groups, group_score):
    x = logits(T, E, dt)
    rng = np.random.default_rng(E)
    for bias in (None, (rng.standard_normal(E) * 0.1).astype(np.float32)):
        for renorm, scale in ((True, 1.0), (False, 2.5)):
            check(capi, x, k, bias, score, groups, top_groups, group_score, renorm, scale, 3 if bias is None else 0)


@pytest.mark.parametrize("T,E,k,groups,top_groups", [(16384, 256, 8, 8, 4), (20000, 64, 6, 1, 1), (5000, 1024, 4, 8, 2), (8191, 128, 16, 4, 2)])
def test_many_tokens(capi, T, E, k, groups, top_groups):
    """Enough tokens that some neighbours' scores lie closer to one another than 32 bits tell."""
    bias = (np.random.default_rng(1).standard_normal(E) * 0.1).astype(np.float32)
    check(capi, logits(T, E), k, bias, "sigmoid", groups, top_groups, "top2", True, 2.5)
    check(capi, logits(T, E, seed=1), k, None, "softmax", groups, top_groups, "max", False, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_nearer_than_32_bits_tell(capi, score):
    """Neighbouring floats as logits, at every size: their scores are equal in 32 bits and are told apart; equal logits go to the lower index."""
    rng = np.random.default_rng(3)
    x = np.empty((400, 64), np.float32)
    for t in range(400):
        base = np.float32(rng.uniform(-6, 6))
        steps = rng.integers(-3, 4, 64)
        row = np.full(64, base, np.float32)
        for i, n in enumerate(steps):
            for _ in range(abs(n)):
                row[i] = np.nextafter(row[i], np.float32(np.inf if n > 0 else -np.inf), dtype=np.float32)
        x[t] = row
    check(capi, torch.from_numpy(x), 6, None, score, 1, 1, "max", True, 1.0)
    check(capi, torch.from_numpy(x), 6, None, score, 8, 2, "top2", True, 1.0)
    # a bias that all but undoes the differences
    s = 1.0 / (1.0 + np.exp(-np.linspace(-2, 2, 64)))
    y = np.tile(np.linspace(-2, 2, 64).astype(np.float32), (50, 1)) + rng.integers(-2, 3, (50, 64)).astype(np.float32) * 1e-7
    check(capi, torch.from_numpy(y.astype(np.float32)), 8, (-s).astype(np.float32), "sigmoid", 1, 1, "max", False, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_far_apart_and_infinite_logits(capi, score):
    """Scores that are zero or one in 32 bits, minus infinity among the logits, biases far larger than the scores."""
    x = logits(64, 64, seed=5, spread=60.0)
    x[3, 7], x[4, :40], x[5, 1] = -np.inf, -np.inf, -1e30
    bias = (np.random.default_rng(2).standard_normal(64) * 100).astype(np.float32)
    for b in (None, bias):
        check(capi, x, 6, b, score, 1, 1, "max", False, 1.0)
        check(capi, x, 6, b, score, 8, 4, "top2", False, 1.0)


@pytest.mark.parametrize("E,k,groups,top", [(33, 11, 3, 1), (33, 3, 11, 1), (40, 8, 1, 1), (45, 15, 3, 1)])
def test_biases_of_minus_infinity(capi, E, k, groups, top):
    """Experts that a bias takes out are chosen last, by their index, and nothing behind the last expert is."""
    x = logits(50, E, seed=4)
    bias = np.zeros(E, np.float32)
    bias[E // 2:] = -np.inf
    for score in ("softmax", "sigmoid"):
        check(capi, x, k, bias, score, groups, top, "max", False, 1.0)
        check(capi, x, k, np.full(E, -np.inf, np.float32), score, groups, top, "max", False, 1.0)


@pytest.mark.parametrize("E,k,groups,top_groups", [(8, 1, 1, 1), (64, 1, 1, 1), (64, 6, 8, 3), (34, 1, 2, 2), (200, 8, 1, 1), (300, 3, 4, 4)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_equal_experts_in_front_of_a_better_one(capi, E, k, groups, top_groups, dt):
    """The last choice and the next expert have one logit, and one behind them is better by less than 32 bits tell: scores that are one in 32 bits, and neighbouring floats."""
    g = torch.Generator().manual_seed(E + k)
    values = torch.tensor([18.0, 20.0, 24.0, 30.0, 45.0])
    x = values[torch.randint(0, 5, (300, E), generator=g)]
    x[:40] = 20.0
    x[torch.arange(40), torch.randint(2, E, (40,), generator=g)] = 25.0
    x[40] = 20.0
    near = torch.full((100, E), 1.0)
    near[torch.arange(100), torch.randint(2, E, (100,), generator=g)] = 1.0 + 2.0 ** -23
    bias = (np.random.default_rng(E).integers(0, 2, E) * 2.0 ** -24).astype(np.float32)
    for score in ("sigmoid", "softmax"):
        for b in (None, bias):
            check(capi, x.to(torch.float32 if dt == "f32" else torch.bfloat16), k, b, score, groups, top_groups, "max", False, 1.0)
            if dt == "f32":
                check(capi, near, k, b, score, groups, top_groups, "top2", False, 1.0)


def test_weights_of_scores_that_32_bits_do_not_hold(capi):
    """The chosen scores are zero in 32 bits, all of them equal or told apart by 64: divided by their sum they are ordinary numbers."""
    x = torch.full((40, 64), -200.0)
    x[20:] += torch.randn(20, 64, generator=torch.Generator().manual_seed(3))
    for groups in (1, 4):
        check(capi, x, 6, None, "sigmoid", groups, groups, "max", True, 1.0)
    # a softmax whose bias chooses experts far below the largest logit
    bias = np.zeros(64, np.float32)
    bias[10:20] = 2.0
    y = logits(40, 64, seed=6)
    y[:, 10:20] -= 150.0
    check(capi, y, 6, bias, "softmax", 1, 1, "max", True, 1.0)
    y[:, 10:20] = y[0, 10]
    check(capi, y, 6, bias, "softmax", 1, 1, "max", True, 2.5)
    # of minus infinity: zero
    y[:, 10:20] = -np.inf
    check(capi, y, 6, bias, "softmax", 1, 1, "max", False, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_nans_rank_last(capi, score, groups):
    """Whatever the logits hold, the ids of a token are distinct and in range."""
    T, E, k = 40, 32, 6
    x = logits(T, E, seed=9)
    x[0], x[1, 3], x[2, :] = np.nan, np.nan, np.inf
    x[3, 5], x[4, :30], x[5, :] = np.inf, np.nan, -np.inf
    ids, w = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, capi.make_moe_gate(x.cuda(), k, ids, w, score=score, num_groups=groups, topk_groups=groups, group_score="top2")))
    got = ids.cpu().numpy()
    assert ((got >= 0) & (got < E)).all() and all(len(set(r)) == k for r in got.tolist())
    assert got[0].tolist() == list(range(k)) and w[0].isnan().all()
    if score == "sigmoid":
        assert 3 not in got[1] and w[1].isfinite().all()
        assert got[2].tolist() == list(range(k)) and got[5].tolist() == list(range(k))
        assert got[3][0] == 5
        assert set(got[4][:2]) == {30, 31} and got[4][2:].tolist() == [0, 1, 2, 3]
    want = gate(x[6:].double().numpy(), k, score, None, groups, groups, "top2")
    assert np.array_equal(got[6:], want[0])


def test_no_tokens_give_zero_counts(capi):
    counts = torch.full((8,), 5, dtype=torch.int32, device="cuda")
    d = capi.make_moe_gate(torch.zeros(0, 8, device="cuda"), 2, torch.zeros(0, 2, dtype=torch.int32, device="cuda"), expert_counts=counts)
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, d))
    assert (counts == 0).all()


def test_host_arrays(capi):
    x = logits(50, 16)
    bias = np.linspace(-1, 1, 16).astype(np.float32)
    ids, w, counts, rows = np.zeros((50, 3), np.int32), np.zeros((50, 3), np.float32), np.zeros(16, np.int32), np.zeros((50, 3), np.int32)
    capi.check(capi.lib.b200dnn_moe_gate(C.byref(capi.make_moe_gate(x.numpy(), 3, ids, w, bias=bias, score="sigmoid", expert_counts=counts, slot_to_row=rows)), None))
    want = gate(x.numpy(), 3, "sigmoid", bias)
    assert np.array_equal(ids, want[0]) and np.array_equal(counts, want[2]) and np.array_equal(rows, want[3])
    np.testing.assert_allclose(w, want[1], rtol=2.0 ** -19)


def test_plain_softmax_is_the_simpler_routers(capi):
    """Without bias and groups, the ids of b200dnn_moe_route (which compares in 32 bits: on logits whose scores these tell apart)."""
    x = torch.from_numpy(np.random.default_rng(0).permuted(np.tile(np.linspace(-3, 3, 64, dtype=np.float32), (500, 1)), axis=1)).cuda()
    got = [[torch.zeros(500, 6, dtype=torch.int32, device="cuda"), torch.zeros(500, 6, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda"),
            torch.zeros(500, 6, dtype=torch.int32, device="cuda")] for _ in range(2)]
    st = torch.cuda.current_stream().cuda_stream
    capi.check(capi.lib.b200dnn_moe_route(x.data_ptr(), 500, 64, 6, 1, *(t.data_ptr() for t in got[0]), st))
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, capi.make_moe_gate(x, 6, got[1][0], got[1][1], expert_counts=got[1][2], slot_to_row=got[1][3])))
    for i in (0, 2, 3):
        assert torch.equal(got[0][i], got[1][i])
    torch.testing.assert_close(got[0][1], got[1][1], rtol=2.0 ** -19, atol=0)
