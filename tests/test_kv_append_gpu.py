"""GPU tests of b200dnn_kv_append against the formula in 64 bits.  Tolerances: a rotated element is two products and a sum in f32 of |a|, |b| <= size: four half steps
of size (2^-22 size); the rounding to bf16 adds 2^-8 of the value (and of that error); a code of an s8 row is off by half a step of the row, and by what its scale is
off: 2^-22 size / 127 and the two roundings of a division and its clamp, 2^-23 of itself."""
import math

import pytest
import torch

from serving import BF16_HALF, Cache, rotated, run, tables

pytestmark = pytest.mark.gpu
DT = dict(bf16=torch.bfloat16, f32=torch.float32)


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


def inputs(g, T, heads, kv_heads, dim, dt, fused=True, pad=0):
    """q, k, v: columns of one matrix, or tensors of their own whose rows lie `pad` elements further apart."""
    if fused:
        x = torch.randn(T, heads + 2 * kv_heads, dim, generator=g, device="cuda").to(DT[dt])
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return [torch.randn(T, n, dim + pad, generator=g, device="cuda").to(DT[dt])[..., :dim] for n in (heads, kv_heads, kv_heads)]


def check(cache, q_out, q, k, v, slots, positions, cos, sin, interleaved, q_before, bits):
    """Every row of a token that has a slot within its tolerance, every other byte as it was."""
    on = slots >= 0
    pages, offs = slots[on] // cache.page, slots[on] % cache.page
    f32 = q_out is not None and q_out.dtype == torch.float32

    def turned(x):
        return rotated(x[on].double(), positions[on], cos, sin, interleaved) if cos is not None else (x[on].double(), torch.zeros_like(x[on].double()))
    if q_out is not None:
        want, size = turned(q)
        tol = 2.0 ** -22 * size + (0 if f32 else BF16_HALF * (want.abs() + size * 2.0 ** -22))
        assert (q_out[on].double() - want).abs().le(tol).all()
        assert torch.equal(q_out[~on].reshape(-1).view(torch.uint8), q_before[~on].reshape(-1).view(torch.uint8))
    for which, (want, size) in enumerate((turned(k), (v[on].double(), torch.zeros_like(v[on].double())))):
        err = 2.0 ** -22 * size
        got = cache.rows(which, pages, offs)
        if cache.dt == "s8":
            scale = cache.scale[which][pages, offs].double()
            exact = (want.abs().amax(-1) / 127.0).clamp(min=1e-10)
            assert ((scale - exact).abs() <= 2.0 ** -22 * size.amax(-1) / 127 + 2.0 ** -22 * exact).all()
            assert ((got - want).abs() <= scale[..., None] * (0.5 + 2.0 ** -15) + err).all()
        else:
            assert ((got - want).abs() <= err + BF16_HALF * (want.abs() + err)).all()
    # the cache's other rows
    for t in cache.kv + [s for s in cache.scale if s is not None]:
        t[pages, offs] = 0
    for now, before, t in zip(cache.bits(), bits, cache.kv + [s for s in cache.scale if s is not None]):
        was = before.view(t.dtype).view(t.shape).clone()
        was[pages, offs] = 0
        assert torch.equal(now, was.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("T", [1, 7, 130])
@pytest.mark.parametrize("cache_dt", ["bf16", "s8"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim,rot,interleaved,page,layout", [
    (32, 8, 128, 128, False, 16, "tokens"), (12, 12, 80, 32, True, 24, "heads"), (4, 1, 64, 64, True, 1, "tokens"), (5, 1, 96, 48, False, 7, "heads"),
    (8, 2, 256, 256, False, 128, "tokens"), (3, 3, 40, 40, False, 16, "tokens"), (2, 1, 72, 16, False, 16, "heads"), (6, 2, 33, 30, True, 5, "tokens"), (2, 2, 1, 0, False, 16, "tokens"),
    (0, 4, 128, 64, False, 32, "heads"), (71, 1, 64, 32, False, 64, "tokens")])
def test_forms(capi, T, cache_dt, dt, heads, kv_heads, dim, rot, interleaved, page, layout):
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + dim)
    cache = Cache(T // page + 3, page, kv_heads, dim, cache_dt, layout)
    q, k, v = inputs(g, T, heads, kv_heads, dim, dt)
    slots = torch.randperm((T // page + 3) * page, generator=g, device="cuda")[:T].clone()
    slots[3::5] = -1
    positions = torch.randint(0, 500, (T,), generator=g, device="cuda", dtype=torch.int32)
    positions[3::5] = -9            # (of padding: not looked at)
    cos, sin = tables(500, rot) if rot else (None, None)
    q_out = torch.randn(T, heads, dim, generator=g, device="cuda").to(DT[dt]) if heads else None
    before = q_out.clone() if heads else None
    bits = cache.bits()
    d = capi.make_kv_append(cache.desc(capi), k, v, slots, q=q if heads else None, q_out=q_out, positions=positions if rot else None, cos=cos, sin=sin, interleaved=interleaved)
    capi.check(run(capi, capi.lib.b200dnn_kv_append, d))
    check(cache, q_out, q, k, v, slots, positions, cos, sin, interleaved, before, bits)


@pytest.mark.parametrize("cache_dt", ["bf16", "s8"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("where", ["q", "k", "v", "q_out", "cache", "tables"])
def test_odd_strides_and_addresses(capi, where, dt, cache_dt):
    """One operand at a time whose rows start on no vector's boundary."""
    g = torch.Generator(device="cuda").manual_seed(11)
    T, heads, kv_heads, dim, page = 33, 6, 2, 64, 16
    cache = Cache(4, page, kv_heads, dim, cache_dt, "tokens", pad=3 if where == "cache" else 0)
    q, k, v = inputs(g, T, heads, kv_heads, dim, dt, fused=False)
    odd = inputs(g, T, heads, kv_heads, dim, dt, fused=False, pad=1)
    q, k, v = odd[0] if where == "q" else q, odd[1] if where == "k" else k, odd[2] if where == "v" else v
    slots = torch.randperm(4 * page, generator=g, device="cuda")[:T].clone()
    slots[7] = -1
    positions = torch.arange(T, device="cuda", dtype=torch.int32)
    cos, sin = tables(64, 64, pad=1 if where == "tables" else 0)
    q_out = torch.zeros(T, heads, dim + (1 if where == "q_out" else 0), device="cuda").to(DT[dt])[..., :dim]
    before, bits = q_out.clone(), cache.bits()
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), k, v, slots, q=q, q_out=q_out, positions=positions, cos=cos, sin=sin)))
    check(cache, q_out, q, k, v, slots, positions, cos, sin, False, before, bits)


@pytest.mark.parametrize("dim,rot,interleaved", [(128, 128, False), (128, 64, True), (50, 20, False)])
def test_queries_rotated_in_place(capi, dim, rot, interleaved):
    g = torch.Generator(device="cuda").manual_seed(3)
    T = 40
    q, k, v = inputs(g, T, 8, 2, dim, "bf16")
    caches = [Cache(4, 16, 2, dim, "bf16") for _ in range(2)]
    slots, positions = torch.arange(T, device="cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    cos, sin = tables(T, rot)
    apart = torch.zeros(T, 8, dim, dtype=torch.bfloat16, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(caches[0].desc(capi), k, v, slots, q=q, q_out=apart, positions=positions, cos=cos, sin=sin, interleaved=interleaved)))
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(caches[1].desc(capi), k, v, slots, q=q, positions=positions, cos=cos, sin=sin, interleaved=interleaved)))
    assert torch.equal(apart, q)
    assert all(torch.equal(a, b) for a, b in zip(caches[0].bits(), caches[1].bits()))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 60])
def test_s8_rows_are_the_librarys_own_quantisation(capi, dt, dim):
    """Without a rotation the codes and scales of the values, and of the keys, are those of b200dnn_quant_per_token, also with zeros and non-finite elements."""
    g = torch.Generator(device="cuda").manual_seed(5)
    T, H = 64, 3
    _, k, v = inputs(g, T, 1, H, dim, dt, fused=False)
    v[3], v[5, 1, 7], v[6, 2, 9], v[8] = 0, math.inf, math.nan, 1e-30
    k[9, 0] = math.nan
    k[11] *= 1e20
    cache = Cache(4, 16, H, dim, "s8", "heads")
    slots = torch.randperm(64, generator=g, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), k, v, slots)))
    for which, x in enumerate((k, v)):
        rows = x.contiguous().view(T * H, dim)
        codes, scale = torch.zeros(T * H, dim, dtype=torch.int8, device="cuda"), torch.zeros(T * H, device="cuda")
        capi.check(capi.lib.b200dnn_quant_per_token(rows.data_ptr(), capi.DT[dt], T * H, dim, dim, codes.data_ptr(), dim, scale.data_ptr(), capi.DT["f32"], torch.cuda.current_stream().cuda_stream))
        assert torch.equal(cache.kv[which][slots // 16, slots % 16], codes.view(T, H, dim))
        assert torch.equal(cache.scale[which][slots // 16, slots % 16], scale.view(T, H))


def test_non_finite_rows_pass(capi):
    """A NaN or an infinity stays where it is (with its partner) and touches no other element."""
    T, dim = 4, 64
    k = torch.ones(T, 1, dim, dtype=torch.bfloat16, device="cuda")
    k[1, 0, 3], k[2, 0, 40] = math.nan, math.inf
    cache = Cache(1, 16, 1, dim, "bf16")
    cos, sin = tables(8, 64)
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), k, k.clone(), torch.arange(T, device="cuda"), positions=torch.full((T,), 3, dtype=torch.int32, device="cuda"),
                                                                      cos=cos, sin=sin)))
    bad = ~cache.kv[0][0, :T, 0].float().isfinite()
    assert bad[1].nonzero()[:, 0].tolist() == [3, 35] and bad[2].nonzero()[:, 0].tolist() == [8, 40] and not bad[0].any() and not bad[3].any()
    same = (cache.kv[1][0, :T] == k) | (cache.kv[1][0, :T].isnan() & k.isnan())
    assert same.all()


@pytest.mark.parametrize("cache_dt,dim", [("bf16", 64), ("s8", 64), ("bf16", 50)])
def test_indices_out_of_range_are_reported_and_leave_the_token_out(capi, cache_dt, dim):
    g = torch.Generator(device="cuda").manual_seed(1)
    T = 6
    q, k, v = inputs(g, T, 2, 1, dim, "bf16")
    cos, sin = tables(10, 32)
    good = torch.arange(T, device="cuda")
    for slots, positions in (([0, 1, 64, 3, 4, 5], [0] * 6), ([0, 1, 1 << 40, 3, 4, 5], [0] * 6), ([0, 1, 2, 3, 4, 5], [0, 1, 10, 3, 4, 5]), ([0, 1, 2, 3, 4, 5], [0, 1, -1, 3, 4, 5])):
        cache = Cache(4, 16, 1, dim, cache_dt)
        slots, positions = torch.tensor(slots, device="cuda"), torch.tensor(positions, dtype=torch.int32, device="cuda")
        q_out = torch.full((T, 2, dim), 5.0, dtype=torch.bfloat16, device="cuda")
        before, bits = q_out.clone(), cache.bits()
        rc = run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), k, v, slots, q=q, q_out=q_out, positions=positions, cos=cos, sin=sin))
        assert rc == capi.FAILURE and "out of range" in capi.last_error()
        assert capi.lib.b200dnn_stream_status(torch.cuda.current_stream().cuda_stream) == capi.SUCCESS      # told once
        seen = good.clone()
        seen[2] = -1
        positions[2] = 0
        check(cache, q_out, q, k, v, seen, positions, cos, sin, False, before, bits)


def test_host_arrays(capi):
    """Everything but the cache may lie in host memory."""
    g = torch.Generator(device="cuda").manual_seed(2)
    T, dim = 9, 64
    q, k, v = (t.contiguous() for t in inputs(g, T, 4, 2, dim, "bf16", fused=False))
    slots, positions = torch.randperm(32, generator=g, device="cuda")[:T], torch.arange(T, device="cuda", dtype=torch.int32)
    cos, sin = tables(16, 64)
    caches = [Cache(2, 16, 2, dim, "s8") for _ in range(2)]
    outs = [torch.zeros(T, 4, dim, dtype=torch.bfloat16, device=where) for where in ("cuda", "cpu")]
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(caches[0].desc(capi), k, v, slots, q=q, q_out=outs[0], positions=positions, cos=cos, sin=sin)))
    capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(caches[1].desc(capi), k.cpu(), v.cpu(), slots.cpu(), q=q.cpu(), q_out=outs[1], positions=positions.cpu(), cos=cos.cpu(),
                                                                      sin=sin.cpu())))
    assert torch.equal(outs[0].cpu(), outs[1]) and all(torch.equal(a, b) for a, b in zip(caches[0].bits(), caches[1].bits()))
    host = Cache(2, 16, 2, dim, "bf16", device="cpu")
    rc = run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(host.desc(capi), k, v, slots))
    assert rc == capi.UNIMPLEMENTED and "device memory" in capi.last_error()


def test_a_descriptor_of_another_device_is_refused(capi):
    k = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache, slots = Cache(1, 16, 1, 64, "bf16"), torch.arange(2, device="cuda")
    d = capi.make_kv_append(cache.desc(capi), k, k, slots)
    assert d.device == torch.cuda.current_device() + 1
    assert capi.make_kv_append(cache.desc(capi), k, k, slots.cpu()).device == 0
    d.device += 1
    assert run(capi, capi.lib.b200dnn_kv_append, d) == capi.FAILURE and "current one" in capi.last_error()
    d.device = -3
    assert run(capi, capi.lib.b200dnn_kv_append, d) == capi.FAILURE
    d.device = 0
    capi.check(run(capi, capi.lib.b200dnn_kv_append, d))
