"""GPU tests of b200dnn_paged_attention against the formula in 64 bits on what the cache holds; the tolerance is derived in serving.attention (a bf16 output adds its
own rounding, an f32 one half a step of f32)."""
import math

import pytest
import torch

from serving import BF16_HALF, F32_HALF, Cache, attention, run, stream

pytestmark = pytest.mark.gpu
DT = dict(bf16=torch.bfloat16, f32=torch.float32)


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


def filled(g, lens, heads, dim, dt, page, layout="tokens", pad=0, spread=1.0, cols=None):
    """A cache that holds sequences of these lengths on pages in no order (every other row stays a NaN), and its table; unused entries name no page."""
    need = [-(-max(0, n) // page) for n in lens]
    cache = Cache(sum(need) + 1, page, heads, dim, dt, layout, pad)
    order = torch.randperm(sum(need) + 1, generator=g, device="cuda").to(torch.int32)
    table, at = torch.full((len(lens), cols or max(need + [1])), -5, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        if n > 0:
            j = torch.arange(n, device="cuda")
            for which in (0, 1):
                cache.put(which, table[i].long()[j // page], j % page, torch.randn(n, heads, dim, generator=g, device="cuda", dtype=torch.float64) * spread)
    return cache, table


def check(capi, cache, table, lens, q, out="bf16", lse=True, out_pad=0, status=None, **kw):
    B, H, D = q.shape
    lens_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = torch.full((B, H, D + out_pad), 9.0, device="cuda").to(DT[out])[..., :D]
    ls = torch.full((B, H), 9.0, device="cuda") if lse else None
    d = capi.make_paged_attention(cache.desc(capi), q, o, table, lens_dev, lse=ls, **kw)
    capi.check(run(capi, capi.lib.b200dnn_paged_attention, d))
    want, wl, tol, ltol = attention(q, cache, table, lens_dev, **kw)
    tol = tol + (BF16_HALF if out == "bf16" else F32_HALF) * (want.abs() + tol)
    for i, n in enumerate(lens):
        if n < 0:
            assert (o[i] == 9).all() and (ls is None or (ls[i] == 9).all())
            continue
        off = (o[i].double() - want[i]).abs()
        assert (off <= tol[i]).all(), (i, n, float((off - tol[i]).max()), int((~(off <= tol[i])).sum()))
        if ls is not None:
            assert torch.equal(ls[i].double(), wl[i]) if n == 0 else ((ls[i].double() - wl[i]).abs() <= ltol[i]).all(), (i, n)
    return o, ls


def queries(g, B, H, D, pad=0, spread=1.0):
    return (torch.randn(B, H, D + pad, generator=g, device="cuda") * spread).to(torch.bfloat16)[..., :D]


LENS = [1, 0, 17, 16, 300, -1, 15, 64, 63, 65, 129, 1000]


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [
    (32, 8, 128, 16, "tokens"), (12, 12, 80, 24, "heads"), (16, 1, 64, 1, "tokens"), (40, 8, 96, 7, "heads"), (8, 2, 256, 128, "tokens"), (9, 1, 128, 64, "heads"),
    (17, 1, 64, 16, "tokens"), (64, 2, 128, 32, "tokens"), (71, 1, 64, 16, "heads"), (24, 2, 192, 16, "tokens"), (3, 3, 40, 16, "tokens"), (4, 2, 72, 16, "heads"), (4, 2, 33, 5, "tokens"),
    (2, 1, 1, 3, "tokens"), (4, 4, 16, 16, "tokens"), (6, 2, 32, 16, "tokens"), (5, 5, 48, 300, "tokens"), (8, 4, 112, 16, "heads")])
def test_forms(capi, dt, heads, kv_heads, dim, page, layout):
    g = torch.Generator(device="cuda").manual_seed(dim * 100 + heads)
    cache, table = filled(g, LENS, kv_heads, dim, dt, page, layout)
    check(capi, cache, table, LENS, queries(g, len(LENS), heads, dim))


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=16), dict(window=100), dict(window=5000), dict(softcap=30.0), dict(softcap=1.5, window=33), dict(scale=0.31), dict(scale=-0.1),
                                dict(sinks=0.5), dict(sinks=60.0, window=70), dict(sinks=-math.inf)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (12, 12, 80), (20, 1, 64), (6, 2, 50)])
def test_windows_caps_scales_and_sinks(capi, dt, out, kw, heads, kv_heads, dim):
    g = torch.Generator(device="cuda").manual_seed(dim)
    kw = dict(kw)
    if "sinks" in kw:
        kw["sinks"] = torch.randn(heads, generator=g, device="cuda") + kw["sinks"]
    cache, table = filled(g, LENS, kv_heads, dim, dt, 16)
    check(capi, cache, table, LENS, queries(g, len(LENS), heads, dim), out=out, **kw)


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("lens", [[20000], [5000, 3, 9001], [70000, 0, 1], [1] * 300, [33] * 1000, list(range(700)), [2048] * 5 + [1] * 60, [-1] * 7, [0] * 5, [4096, -1] * 20])
def test_lengths(capi, dt, lens):
    """One long sequence split over the device, many short ones, both together, nothing but padding."""
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    cache, table = filled(g, lens, 2, 128, dt, 32)
    check(capi, cache, table, lens, queries(g, len(lens), 8, 128))


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (10, 5), (22, 11), (32, 16), (20, 20), (72, 6)])
@pytest.mark.parametrize("lens", [[900] * 40, [3, 20000, 0, 64, 129], list(range(0, 3000, 37))])
def test_numbers_of_rows(capi, dt, heads, kv_heads, lens):
    """Rows of a sequence that go side by side, eight at a time and where eight do not divide them, with sequences that begin and end inside every share of the work."""
    g = torch.Generator(device="cuda").manual_seed(kv_heads)
    cache, table = filled(g, lens, kv_heads, 64, dt, 16)
    check(capi, cache, table, lens, queries(g, len(lens), heads, 64))


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("spread", [0.0, 8.0, 40.0])
def test_peaked_and_flat_softmax(capi, dt, spread):
    """Scores far apart (the running maximum moves again and again), and all equal."""
    g = torch.Generator(device="cuda").manual_seed(7)
    lens = [3000, 70, 1]
    cache, table = filled(g, lens, 2, 128, dt, 16, spread=1.0)
    # the scores grow along the sequence: every block raises the maximum
    j = torch.arange(3000, device="cuda")
    grow = torch.linspace(0, 1, 3000, dtype=torch.float64, device="cuda")[:, None, None]
    cache.put(0, table[0].long()[j // 16], j % 16, grow * torch.ones(3000, 2, 128, dtype=torch.float64, device="cuda") * 2 + torch.randn(3000, 2, 128, generator=g, device="cuda", dtype=torch.float64) * 0.1)
    check(capi, cache, table, lens, queries(g, 3, 8, 128, spread=spread).abs())


@pytest.mark.parametrize("sizes", [1e-30, 1e-6, 1e6, 1e30])
@pytest.mark.parametrize("dt", ["bf16", "s8"])
def test_values_and_queries_of_any_magnitude(capi, dt, sizes):
    """Values (and for s8 their scales) of any size, all alike and very different from key to key; queries as far from one as the keys are the other way."""
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [257, 40]
    cache, table = filled(g, lens, 1, 64, dt, 16)
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        pages, offs = table[i].long()[j // 16], j % 16
        x = torch.randn(n, 1, 64, generator=g, device="cuda", dtype=torch.float64)
        cache.put(1, pages, offs, x * sizes * (10.0 ** (-4.0 * (j % 3 == 1).double()))[:, None, None] if i else x * sizes)
        cache.put(0, pages, offs, torch.randn(n, 1, 64, generator=g, device="cuda", dtype=torch.float64) * max(1e-6, min(1e6, 1 / sizes)))
    q = queries(g, 2, 4, 64, spread=max(1e-6, min(1e6, sizes)))
    check(capi, cache, table, lens, q, out="f32")


@pytest.mark.parametrize("dt", ["bf16", "s8"])
@pytest.mark.parametrize("where", ["q", "out", "cache"])
def test_odd_strides(capi, where, dt):
    g = torch.Generator(device="cuda").manual_seed(13)
    lens = [100, 40, 0, 7]
    cache, table = filled(g, lens, 2, 64, dt, 16, pad=3 if where == "cache" else 0)
    check(capi, cache, table, lens, queries(g, 4, 8, 64, pad=1 if where == "q" else 0), out_pad=1 if where == "out" else 0)


def test_queries_that_are_part_of_a_wider_matrix(capi):
    g = torch.Generator(device="cuda").manual_seed(13)
    lens = [100, 40, 0, 7]
    cache, table = filled(g, lens, 2, 64, "bf16", 16)
    wide = torch.randn(4, 12, 64, generator=g, device="cuda").to(torch.bfloat16)
    wide_table = torch.full((4, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    a, _ = check(capi, cache, wide_table[:, :table.shape[1]], lens, wide[:, 2:10])
    b, _ = check(capi, cache, wide_table, lens, wide[:, 2:10].contiguous())
    assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [128, 50])
def test_non_finite_values_that_are_seen(capi, dim):
    """A NaN value among the visible ones reaches its own column alone; an infinite score makes the row a NaN, a score of minus infinity takes its key out."""
    g = torch.Generator(device="cuda").manual_seed(4)
    lens = [200, 200, 200, 30]
    cache, table = filled(g, lens, 1, dim, "bf16", 16)
    q = queries(g, 4, 4, dim).abs()
    j = 77
    cache.kv[1][table[0, j // 16], j % 16, 0, 5] = math.nan
    cache.kv[0][table[1, j // 16], j % 16, 0, 5] = math.inf
    cache.kv[0][table[2, j // 16], j % 16, 0, 5] = -math.inf
    for n in range(30):
        cache.kv[0][table[3, n // 16], n % 16, 0, 5] = -math.inf
    o = torch.zeros(4, 4, dim, dtype=torch.bfloat16, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), q, o, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))))
    bad = o[0].isnan()
    assert bad[:, 5].all() and bad.sum() == 4
    assert o[1].isnan().all()
    assert o[2].isfinite().all()
    assert (o[3] == 0).all()             # no key left: a row without keys
    at = torch.arange(200, device="cuda")
    at = at[at != j]
    k, v = (cache.rows(w, table[2].long()[at // 16], at % 16)[:, 0] for w in (0, 1))
    p = torch.softmax(q[2].double() @ k.T * dim ** -0.5, -1)
    assert ((p @ v - o[2].double()).abs() <= BF16_HALF * (p @ v).abs() + 2.0 ** -12 * (p @ v.abs())).all()


@pytest.mark.parametrize("dt,dim", [("bf16", 128), ("s8", 128), ("bf16", 50)])
def test_pages_and_lengths_out_of_range_are_reported(capi, dt, dim):
    g = torch.Generator(device="cuda").manual_seed(6)
    lens = [100, 64, 90]
    cache, table = filled(g, lens, 2, dim, dt, 16)
    q = queries(g, 3, 4, dim)
    good, _ = check(capi, cache, table, lens, q)
    entry = capi.lib.b200dnn_paged_attention
    for spoil in ("negative", "beyond", "length"):
        t, n = table.clone(), list(lens)
        if spoil == "negative":
            t[1, 2] = -1
        elif spoil == "beyond":
            t[1, 2] = cache.kv[0].shape[0]
        else:
            n[1] = 16 * table.shape[1] + 1
        o = torch.zeros(3, 4, dim, dtype=torch.bfloat16, device="cuda")
        rc = run(capi, entry, capi.make_paged_attention(cache.desc(capi), q, o, t, torch.tensor(n, dtype=torch.int32, device="cuda")))
        assert rc == capi.FAILURE and "out of range" in capi.last_error(), spoil
        assert capi.lib.b200dnn_stream_status(stream()) == capi.SUCCESS
        assert torch.equal(o[0], good[0]) and torch.equal(o[2], good[2])


def test_repeated_calls_give_the_same_bits(capi):
    g = torch.Generator(device="cuda").manual_seed(8)
    lens = [30000, 11, 4000, 0, 900]
    cache, table = filled(g, lens, 4, 128, "bf16", 16)
    q = queries(g, 5, 16, 128)
    first, lse = check(capi, cache, table, lens, q)
    for _ in range(20):
        o, ls = torch.zeros_like(first), torch.zeros_like(lse)
        capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), q, o, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), lse=ls)))
        assert torch.equal(o, first) and torch.equal(ls, lse)


def test_host_arrays(capi):
    g = torch.Generator(device="cuda").manual_seed(2)
    lens = [50, 3, 0, -1]
    cache, table = filled(g, lens, 2, 64, "s8", 16)
    q, sinks = queries(g, 4, 4, 64), torch.randn(4, generator=g, device="cuda")
    dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    outs, lses = [torch.full((4, 4, 64), 3.0, device=w) for w in ("cuda", "cpu")], [torch.full((4, 4), 3.0, device=w) for w in ("cuda", "cpu")]
    for n, t in ((0, lambda x: x), (1, lambda x: x.cpu())):
        capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), t(q), outs[n], t(table), t(dev), sinks=t(sinks), lse=lses[n])))
    assert torch.equal(outs[0].cpu(), outs[1]) and torch.equal(lses[0].cpu(), lses[1])
