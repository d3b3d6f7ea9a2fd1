"""The serving operators as a program uses them: prompts appended to a paged cache, then decode steps -- queries and keys rotated, the new token appended, attention over the cache, the block's
experts chosen and computed -- captured into a CUDA graph and replayed while positions, slots and lengths move on; and several streams, one descriptor per step."""
import ctypes as C

import numpy as np
import pytest
import torch

from serving import BF16_HALF, Cache, attention, gate, rotated, run, stream, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


class Sequences:
    """Pages handed out to sequences as they grow, as a scheduler does it."""

    def __init__(self, batch, page, cols, seed):
        self.free = np.random.default_rng(seed).permutation(batch * cols).tolist()
        self.table, self.lens, self.page = np.full((batch, cols), -1, np.int32), np.zeros(batch, np.int32), page

    def grow(self, i, n):
        """Slots and positions of n new tokens of sequence i."""
        slots = []
        for p in range(self.lens[i], self.lens[i] + n):
            if p % self.page == 0:
                self.table[i, p // self.page] = self.free.pop()
            slots.append(int(self.table[i, p // self.page]) * self.page + p % self.page)
        at = list(range(self.lens[i], self.lens[i] + n))
        self.lens[i] += n
        return slots, at


@pytest.mark.parametrize("dt,heads,kv_heads,dim,page", [("bf16", 8, 2, 128, 16), ("s8", 12, 4, 64, 24), ("bf16", 6, 2, 40, 5)])
def test_prompts_and_captured_decode_steps(capi, dt, heads, kv_heads, dim, page):
    B, prompts, steps, cols = 4, [37, 1, 64, 5], 20, 24
    g = torch.Generator(device="cuda").manual_seed(dim)
    seqs, cache = Sequences(B, page, cols, 1), Cache(B * cols, page, kv_heads, dim, dt)
    rot = dim // 2
    cos, sin = tables(512, rot)
    new = lambda n, h: torch.randn(n, h, dim, generator=g, device="cuda").to(torch.bfloat16)
    keys, values = [[] for _ in range(B)], [[] for _ in range(B)]
    # the prompts, two calls of several sequences each
    for part in ([0, 1], [2, 3]):
        slots, at, owner = [], [], []
        for i in part:
            s, p = seqs.grow(i, prompts[i])
            slots, at, owner = slots + s, at + p, owner + [i] * len(s)
        k, v, q = new(len(slots), kv_heads), new(len(slots), kv_heads), new(len(slots), heads)
        positions = torch.tensor(at, dtype=torch.int32, device="cuda")
        d = capi.make_kv_append(cache.desc(capi), k, v, torch.tensor(slots, device="cuda"), q=q, positions=positions, cos=cos, sin=sin)
        kr = rotated(k.double(), positions, cos, sin, False)[0]
        capi.check(run(capi, capi.lib.b200dnn_kv_append, d))
        for j, i in enumerate(owner):
            keys[i].append(kr[j])
            values[i].append(v[j].double())
    # decode: fixed buffers, one graph; row B is padding
    n = B + 1
    qkv = torch.zeros(n, heads + 2 * kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    q_out, out = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, heads, dim, device="cuda")
    slots, positions = torch.full((n,), -1, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    table, lens = torch.full((n, cols), -1, dtype=torch.int32, device="cuda"), torch.full((n,), -1, dtype=torch.int32, device="cuda")
    append = capi.make_kv_append(cache.desc(capi), k, v, slots, q=q, q_out=q_out, positions=positions, cos=cos, sin=sin)
    attend = capi.make_paged_attention(cache.desc(capi), q_out, out, table, lens)
    side = torch.cuda.Stream()

    def step():
        capi.check(capi.lib.b200dnn_kv_append(C.byref(append), side.cuda_stream))
        capi.check(capi.lib.b200dnn_paged_attention(C.byref(attend), side.cuda_stream))

    side.wait_stream(torch.cuda.current_stream())
    step()                                     # nothing but padding
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(steps):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        for i in range(B):
            s, p = seqs.grow(i, 1)
            slots[i], positions[i] = s[0], p[0]
        table[:B], lens[:B] = torch.from_numpy(seqs.table).cuda(), torch.from_numpy(seqs.lens).cuda()
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kr, qr = (rotated(x.double(), positions, cos, sin, False)[0] for x in (k, q))
        for i in range(B):
            keys[i].append(kr[i])
            values[i].append(v[i].double())
        want, _, tol, _ = attention(q_out[:B], cache, table[:B], lens[:B])
        assert ((out[:B].double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()
        assert (out[B] == 7).all()
        assert ((q_out[:B].double() - qr[:B]).abs() <= BF16_HALF * qr[:B].abs() + 2.0 ** -7 * 2.0 ** -8).all()
    capi.check(capi.lib.b200dnn_stream_status(side.cuda_stream))
    # the cache holds every token's row: rounded to bf16, or within half a step of its row's codes
    for i in range(B):
        at = torch.arange(int(seqs.lens[i]), device="cuda")
        pages = torch.from_numpy(seqs.table[i]).cuda().long()[at // page]
        for which, rows in enumerate((keys[i], values[i])):
            want = torch.stack(rows)
            half = want.abs().amax(-1, keepdim=True) / 127 * 0.5001 if dt == "s8" else BF16_HALF * want.abs() + 2.0 ** -20
            assert ((cache.rows(which, pages, at % page) - want).abs() <= half + 2.0 ** -20).all()


def test_attention_agrees_with_the_dense_operator(capi):
    """The same keys and values through b200dnn_sdpa (dense, one head for every query head)."""
    B, H, n, D = 3, 8, 200, 128
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(B, H, n, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(B, H, 1, D, generator=g, device="cuda").to(torch.bfloat16)
    cache, table = Cache(B * 13, 16, H, D, "bf16", "heads"), torch.randperm(B * 13, generator=g, device="cuda").to(torch.int32).view(B, 13)
    j = torch.arange(n, device="cuda")
    for i in range(B):
        for which, x in enumerate((k, v)):
            cache.put(which, table[i].long()[j // 16], j % 16, x[i].transpose(0, 1).double())
    outs = [torch.zeros(B, H, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    d = capi.SdpaDesc()
    d.batch, d.num_heads, d.seq_len, d.kv_seq_len, d.head_dim = B, H, 1, n, D
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v), ("o_stride", outs[0])):
        setattr(d, name, (C.c_int64 * 4)(*t.stride()))
    d.qkv_dt = d.out_dt = capi.DT["bf16"]
    d.query, d.key, d.value, d.output = q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[0].data_ptr()
    capi.check(run(capi, capi.lib.b200dnn_sdpa, d))
    capi.check(run(capi, capi.lib.b200dnn_paged_attention,
                   capi.make_paged_attention(cache.desc(capi), q[:, :, 0], outs[1][:, :, 0], table, torch.full((B,), n, dtype=torch.int32, device="cuda"))))
    # two bf16 roundings of the result, and the dense operator's of its probabilities (2^-8 of a convex combination of values)
    assert ((outs[0].double() - outs[1].double()).abs() <= 2 * BF16_HALF * (outs[1].double().abs() + v.double().abs().amax(2, keepdim=True) / 8)).all()


def test_routing_drives_the_expert_blocks(capi, oracle):
    """Choice, weights, counts and places of b200dnn_moe_gate through the blocks that take them: rows quantised once and scattered, the experts, the weighted sum."""
    T, H, I, E, k = 96, 128, 64, 8, 3
    rng = np.random.default_rng(0)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
    logits = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).cuda()
    bias = torch.from_numpy((rng.standard_normal(E) * 0.2).astype(np.float32)).cuda()
    ex, keep = (capi.MoeExpert * E)(), []
    for e in range(E):
        w = [torch.from_numpy(rng.integers(-127, 128, s, dtype=np.int8)).cuda() for s in ((H, 2 * I), (I, H))]
        s = [torch.full((n,), 1e-3, device="cuda") for n in (2 * I, H)]
        keep.append((w, s))
        ex[e].w13, ex[e].ldb13, ex[e].w13_scale, ex[e].w2, ex[e].ldb2, ex[e].w2_scale = w[0].data_ptr(), 2 * I, s[0].data_ptr(), w[1].data_ptr(), H, s[1].data_ptr()
    ids, weights = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
    counts, places = torch.zeros(E, dtype=torch.int32, device="cuda"), torch.zeros(T, k, dtype=torch.int32, device="cuda")
    st = stream()
    capi.check(capi.lib.b200dnn_moe_gate(C.byref(capi.make_moe_gate(logits, k, ids, weights, bias=bias, score="sigmoid", num_groups=4, topk_groups=2, group_score="top2", scale=2.5, expert_counts=counts,
                                                                    slot_to_row=places)), st))
    rows, row_scale = torch.zeros(T * k, H, dtype=torch.int8, device="cuda"), torch.zeros(T * k, device="cuda")
    capi.check(capi.lib.b200dnn_quant_per_token_scatter(x.data_ptr(), capi.DT["bf16"], H, H, places.data_ptr(), k, T, rows.data_ptr(), H, row_scale.data_ptr(), st))
    torch.cuda.synchronize()
    n = counts.cpu().numpy()
    experts_out, out = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    capi.check(capi.lib.b200dnn_moe_experts_s8(rows.data_ptr(), H, row_scale.data_ptr(), E, n.ctypes.data, np.arange(E, dtype=np.int32).ctypes.data, ex, H, I, H, 0, capi.ACT["silu_and_mul"],
                                               experts_out.data_ptr(), H, st))
    capi.check(capi.lib.b200dnn_moe_weighted_reduce_rows(experts_out.data_ptr(), H, places.data_ptr(), weights.data_ptr(), T, k, H, capi.DT["bf16"], out.data_ptr(), H, st))
    capi.check(capi.lib.b200dnn_stream_status(st))
    want_ids, want_w, want_n, want_rows = gate(logits.cpu().numpy(), k, "sigmoid", bias.cpu().numpy(), 4, 2, "top2", True, 2.5)
    assert np.array_equal(ids.cpu().numpy(), want_ids) and np.array_equal(n, want_n) and np.array_equal(places.cpu().numpy(), want_rows)
    bits = x.view(torch.int16).cpu().numpy().view(np.uint16)
    ref, _ = oracle.fused_moe(bits, want_ids, weights.cpu().numpy(), [w[0].cpu().numpy() for w, _ in keep], [s[0].cpu().numpy() for _, s in keep], [w[1].cpu().numpy() for w, _ in keep],
                              [s[1].cpu().numpy() for _, s in keep])
    from helpers import assert_bf16_close
    assert_bf16_close(out.view(torch.int16).cpu().numpy().view(np.uint16), ref, max_ulp=1, what="experts", row_atol_frac=2.0 ** -7)


@pytest.mark.parametrize("T,E,S,k", [(1, 4, 0, 2), (32, 64, 2, 6), (64, 255, 1, 3), (300, 16, 1, 4), (200, 300, 0, 5)])
def test_a_layer_routed_by_the_caller(capi, T, E, S, k):
    """b200dnn_moe_layer_routed on the ids and weights of b200dnn_moe_route is b200dnn_moe_layer bit for bit (in all forms of the routing); ids out of range meet the nearest expert."""
    H, I = 128, 64
    rng = np.random.default_rng(E)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
    logits = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).cuda()
    w13, w2 = (torch.from_numpy(rng.integers(-127, 128, (E + S, *s), dtype=np.int8)).cuda() for s in ((H, 2 * I), (I, H)))
    s13, s2 = torch.full((2 * I,), 1e-3, device="cuda"), torch.full((H,), 1e-3, device="cuda")
    ex = (capi.MoeExpert * (E + S))()
    for e in range(E + S):
        ex[e].w13, ex[e].ldb13, ex[e].w13_scale, ex[e].w2, ex[e].ldb2, ex[e].w2_scale = w13[e].data_ptr(), 2 * I, s13.data_ptr(), w2[e].data_ptr(), H, s2.data_ptr()
    st = stream()
    ids, w = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
    capi.check(capi.lib.b200dnn_moe_route(logits.data_ptr(), T, E, k, 1, ids.data_ptr(), w.data_ptr(), None, None, st))
    outs = [torch.zeros(T, H, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    tail = lambda o: (T, E, S, k, ex, H, I, H, 0, capi.ACT["silu_and_mul"], o.data_ptr(), H, st)
    capi.check(capi.lib.b200dnn_moe_layer(x.data_ptr(), H, logits.data_ptr(), *tail(outs[0])))
    capi.check(capi.lib.b200dnn_moe_layer_routed(x.data_ptr(), H, ids.data_ptr(), w.data_ptr(), *tail(outs[1])))
    capi.check(capi.lib.b200dnn_stream_status(st))
    assert torch.equal(outs[0], outs[1])
    far = ids.clone()
    far[ids == E - 1], far[ids == 0] = E + 1000, -5
    capi.check(capi.lib.b200dnn_moe_layer_routed(x.data_ptr(), H, far.data_ptr(), w.data_ptr(), *tail(outs[2])))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2])
    assert capi.lib.b200dnn_moe_layer_routed(x.data_ptr(), H, None, w.data_ptr(), *tail(outs[2])) == capi.FAILURE and "null" in capi.last_error()
    capi.lib.b200dnn_clear_caches()


def test_two_streams_at_once(capi):
    """Calls on streams of their own share no workspace: long and short batches side by side, many times, give what each gives alone."""
    from test_paged_attention_gpu import filled, queries
    g = torch.Generator(device="cuda").manual_seed(1)
    jobs = []
    for lens in ([9000, 30, 2000], [700] * 40):
        cache, table = filled(g, lens, 2, 128, "bf16", 16)
        q, dev = queries(g, len(lens), 8, 128), torch.tensor(lens, dtype=torch.int32, device="cuda")
        alone = torch.zeros_like(q)
        capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), q, alone, table, dev)))
        out = torch.zeros_like(q)
        jobs.append((capi.make_paged_attention(cache.desc(capi), q, out, table, dev), torch.cuda.Stream(), alone, out))
    for _ in range(20):
        for d, _, _, out in jobs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for d, s, _, _ in jobs:
                capi.check(capi.lib.b200dnn_paged_attention(C.byref(d), s.cuda_stream))
        torch.cuda.synchronize()
        for _, _, alone, out in jobs:
            assert torch.equal(alone, out)


def test_graphs_captured_on_one_stream_run_side_by_side(capi):
    """Graphs have scratch of their own: two captured one after the other on a stream, replayed on two streams at once and beside a call on the stream they were captured on, give
    what each call gives alone; a graph's scratch serves later ones when it is gone."""
    from test_paged_attention_gpu import filled, queries
    g = torch.Generator(device="cuda").manual_seed(2)
    home = torch.cuda.Stream()
    jobs = []
    for lens in ([20000, 5], [15000, 100, 9000], [12345]):
        cache, table = filled(g, lens, 2, 64, "bf16", 16)
        q, dev = queries(g, len(lens), 8, 64), torch.tensor(lens, dtype=torch.int32, device="cuda")
        x = torch.randn(2000, 64, generator=g, device="cuda")
        alone, out = torch.zeros_like(q), torch.zeros_like(q)
        gates = []
        for _ in range(2):
            t = [torch.zeros(2000, 4, dtype=torch.int32, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(2000, 4, dtype=torch.int32, device="cuda")]
            gates.append((capi.make_moe_gate(x, 4, t[0], expert_counts=t[1], slot_to_row=t[2]), t))
        capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), q, alone, table, dev)))
        capi.check(run(capi, capi.lib.b200dnn_moe_gate, gates[0][0]))
        jobs.append((capi.make_paged_attention(cache.desc(capi), q, out, table, dev), gates[1][0], (alone, *gates[0][1]), (out, *gates[1][1])))

    def calls(job, st):
        capi.check(capi.lib.b200dnn_paged_attention(C.byref(job[0]), st))
        capi.check(capi.lib.b200dnn_moe_gate(C.byref(job[1]), st))

    for round_ in range(3):
        torch.cuda.synchronize()
        graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
        for job in jobs[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=home):
                calls(job, home.cuda_stream)
                calls(job, home.cuda_stream)
            graphs.append(graph)
        for _ in range(10):
            for job in jobs:
                for t in job[3]:
                    t.zero_()
            torch.cuda.synchronize()
            for _ in range(2):
                for s, graph in zip(streams, graphs):
                    with torch.cuda.stream(s):
                        graph.replay()
                calls(jobs[2], home.cuda_stream)
            torch.cuda.synchronize()
            for job in jobs:
                assert all(torch.equal(a, b) for a, b in zip(job[2], job[3]))
        del graphs, graph


@pytest.mark.parametrize("dt,dim,page", [("bf16", 64, 16), ("s8", 64, 16), ("bf16", 64, 12), ("bf16", 50, 16)])
def test_offsets_beyond_32_bits(capi, dt, dim, page):
    """Pages that lie 1.3 billion elements apart hold and give what adjacent ones do: appended to, read, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(5)
    T, kv_heads, heads, pages, apart = 4 * page - 3, 2, 6, 4, 1_300_000_000
    shape, kind = (pages, page, kv_heads, dim), torch.int8 if dt == "s8" else torch.bfloat16
    far = torch.empty((pages - 1) * apart + 2 * page * kv_heads * dim, dtype=kind, device="cuda")
    k, v = (torch.randn(T, kv_heads, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, heads, dim, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.tensor([[3, 0, 2, 1]], dtype=torch.int32, device="cuda")
    at = torch.arange(T, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    got = []
    for wide in (False, True):
        row = (kv_heads * dim, dim, 1)
        kv = [far.as_strided(shape, (apart, *row), n * page * kv_heads * dim) for n in (0, 1)] if wide else [torch.zeros(shape, dtype=kind, device="cuda") for _ in range(2)]
        scales = [torch.zeros(shape[:3], device="cuda") for _ in range(2)] if dt == "s8" else []
        cache = capi.make_kv_cache(*kv, *scales)
        out = torch.zeros(1, heads, dim, device="cuda")
        capi.check(run(capi, capi.lib.b200dnn_kv_append, capi.make_kv_append(cache, k, v, slots)))
        capi.check(run(capi, capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache, q, out, table, torch.tensor([T], dtype=torch.int32, device="cuda"))))
        got.append((out, *(t.clone() for t in kv), *scales))
    # (of the last page, three tokens were never written)
    written = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    written[table[0, -1].long() * page + torch.arange(page - 3, page, device="cuda")] = False
    assert torch.equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1:], got[1][1:]):
        assert torch.equal(a.flatten(0, 1)[written], b.flatten(0, 1)[written])
