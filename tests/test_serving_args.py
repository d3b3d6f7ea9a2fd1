"""What the serving entry points refuse, and what they make of nothing: checks of the arguments alone, without a GPU."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    return c


def u16(*shape):
    return np.zeros(shape, dtype=np.uint16)


def cache(capi, dt="bf16", dim=64, page=16, heads=2, pages=4):
    if dt == "s8":
        return capi.make_kv_cache(*(np.zeros((pages, page, heads, dim), np.int8) for _ in range(2)), *(np.zeros((pages, page, heads), np.float32) for _ in range(2)))
    return capi.make_kv_cache(u16(pages, page, heads, dim), u16(pages, page, heads, dim))


def append(capi, T=3, **kw):
    c = cache(capi, **kw)
    tab = np.zeros((8, 32), np.float32)
    return capi.make_kv_append(c, u16(T, 2, 64), u16(T, 2, 64), np.zeros(T, np.int64), q=u16(T, 4, 64), q_out=u16(T, 4, 64), positions=np.zeros(T, np.int32), cos=tab, sin=tab)


def attend(capi, B=3, **kw):
    return capi.make_paged_attention(cache(capi, **kw), u16(B, 4, 64), u16(B, 4, 64), np.zeros((B, 2), np.int32), np.zeros(B, np.int32))


def gate(capi, T=3, E=8, k=2, **kw):
    return capi.make_moe_gate(np.zeros((T, E), np.float32), k, np.zeros((T, k), np.int32), **kw)


def refused(capi, entry, desc, text, status=None):
    rc = getattr(capi.lib, entry)(C.byref(desc), None)
    assert rc == (capi.FAILURE if status is None else status) and text in capi.last_error(), (rc, capi.last_error())


def test_struct_layout_matches_header(capi):
    assert C.sizeof(capi.KvCache) == 4 * 4 + 8 + 4 * 8 + 9 * 8
    assert C.sizeof(capi.KvAppendDesc) == C.sizeof(capi.KvCache) + 8 + 4 * 4 + 8 * 8 + 7 * 8 + 2 * 8 + 8 + 2 * 4
    assert C.sizeof(capi.PagedAttentionDesc) == C.sizeof(capi.KvCache) + 4 * 4 + 4 * 8 + 4 * 8 + 8 + 2 * 4 + 2 * 8 + 8 + 2 * 4
    assert C.sizeof(capi.MoeGateDesc) == 10 * 4 + 8 + 6 * 8 + 2 * 4


def test_null_descriptors(capi):
    for entry in ("b200dnn_kv_append", "b200dnn_paged_attention", "b200dnn_moe_gate"):
        assert getattr(capi.lib, entry)(None, None) == capi.FAILURE and "null" in capi.last_error()


@pytest.mark.parametrize("make,entry", [(append, "b200dnn_kv_append"), (attend, "b200dnn_paged_attention")])
def test_cache_refusals(capi, make, entry):
    def bad(text, status=None, dt="bf16", **fields):
        d = make(capi, dt=dt)
        for k, v in fields.items():
            setattr(d.cache, k, v)
        refused(capi, entry, d, text, status)
    d = make(capi); d.cache.dt = capi.DT["f32"]; refused(capi, entry, d, "bf16 or s8", capi.UNIMPLEMENTED)
    bad("must be > 0", page_size=0)
    bad("must be > 0", kv_heads=-2)
    bad("must be > 0", num_pages=0)
    bad("up to 256", capi.UNIMPLEMENTED, head_dim=257)
    bad("null", key=None)
    bad("null", value=None)
    bad("key_scale", dt="s8", key_scale=None)
    bad("scale stride", dt="s8", scale_stride=(C.c_int64 * 3)(32, 2, 0))
    bad("overlap", key_stride=(C.c_int64 * 3)(2048, 128, 63))
    bad("overlap", value_stride=(C.c_int64 * 3)(0, 128, 64))
    bad("2^31", capi.UNIMPLEMENTED, key_stride=(C.c_int64 * 3)(1 << 31, 128, 64))


def test_append_refusals(capi):
    def bad(text, status=None, **fields):
        d = append(capi)
        for k, v in fields.items():
            setattr(d, k, v)
        refused(capi, "b200dnn_kv_append", d, text, status)
    bad(">= 0", num_tokens=-1)
    bad(">= 0", q_heads=-1)
    bad("bf16 or f32", capi.UNIMPLEMENTED, dt=capi.DT["s8"])
    bad("rotary_dim", rotary_dim=7)
    bad("rotary_dim", rotary_dim=66)
    bad("rotary_dim", rotary_dim=-2)
    bad("null", k=None)
    bad("null", slots=None)
    bad("q or q_out", q_out=None)
    bad("strides", k_stride=(C.c_int64 * 2)(128, 63))
    bad("strides", q_out_stride=(C.c_int64 * 2)(0, 64))
    bad("positions", positions=None)
    bad("positions", table_rows=0)
    bad("positions", table_ld=31)
    bad("too many", capi.UNIMPLEMENTED, num_tokens=1 << 33)
    d = append(capi)
    d.q_out = d.q
    d.q_out_stride = (C.c_int64 * 2)(512, 64)
    refused(capi, "b200dnn_kv_append", d, "in place")


def test_attention_refusals(capi):
    def bad(text, status=None, **fields):
        d = attend(capi)
        for k, v in fields.items():
            setattr(d, k, v)
        refused(capi, "b200dnn_paged_attention", d, text, status)
    bad(">= 0", num_seqs=-1)
    bad("multiple", q_heads=3)
    bad("multiple", q_heads=0)
    bad("queries are bf16", capi.UNIMPLEMENTED, q_dt=capi.DT["f32"])
    bad("output is", capi.UNIMPLEMENTED, out_dt=capi.DT["s8"])
    bad("window", window=-1)
    bad("softcap", softcap=-1.0)
    bad("softcap", softcap=float("inf"))
    bad("scale", scale=float("nan"))
    bad("max_pages", max_pages=0)
    bad("max_pages", max_pages=3)
    bad("null", seq_lens=None)
    bad("null", page_table=None)
    bad("strides", q_stride=(C.c_int64 * 2)(256, 1))
    bad("too many", capi.UNIMPLEMENTED, num_seqs=1 << 30)
    bad("2^30", capi.UNIMPLEMENTED, max_pages=1 << 26, page_table_ld=1 << 26)
    d = attend(capi)
    d.out = d.q
    refused(capi, "b200dnn_paged_attention", d, "overlap")


def test_gate_refusals(capi):
    def bad(text, status=None, **fields):
        d = gate(capi)
        for k, v in fields.items():
            setattr(d, k, v)
        refused(capi, "b200dnn_moe_gate", d, text, status)
    bad("num_tokens", num_tokens=-1)
    bad("num_tokens", num_experts=0)
    bad("1024", capi.UNIMPLEMENTED, num_experts=1025, ld=1025)
    bad("score", score=2)
    bad("num_groups", num_groups=3)
    bad("num_groups", num_groups=0)
    bad("num_groups", topk_groups=2)
    bad("num_groups", num_groups=4, topk_groups=0)
    bad("32 groups", capi.UNIMPLEMENTED, num_experts=64, num_groups=64, topk_groups=64, ld=64)
    bad("group_score", group_score=5)
    bad("topk", topk=0)
    bad("topk", topk=9)
    bad("topk", num_groups=4, topk_groups=1, topk=3)
    bad("up to 16", capi.UNIMPLEMENTED, num_experts=32, ld=32, topk=17)
    bad("finite", scale=float("inf"))
    bad("f32 or bf16", capi.UNIMPLEMENTED, logits_dt=capi.DT["s8"])
    bad("null", ids=None)
    bad("ld", ld=7)


def test_nothing_to_do(capi):
    """No token, no sequence: success without a look at the pointers (or at a GPU)."""
    d = append(capi)
    d.num_tokens, d.k, d.slots = 0, None, None
    assert capi.lib.b200dnn_kv_append(C.byref(d), None) == capi.SUCCESS
    d = attend(capi)
    d.num_seqs, d.q = 0, None
    assert capi.lib.b200dnn_paged_attention(C.byref(d), None) == capi.SUCCESS
    d = gate(capi)
    d.num_tokens, d.logits, d.ids = 0, None, None
    assert capi.lib.b200dnn_moe_gate(C.byref(d), None) == capi.SUCCESS


def test_python_helpers_refuse_what_the_descriptor_cannot_say(capi):
    k = u16(4, 16, 2, 64)
    with pytest.raises(ValueError, match="dense"):
        capi.make_kv_cache(u16(4, 16, 2, 128)[..., ::2], k)
    with pytest.raises(ValueError, match="one shape"):
        capi.make_kv_cache(k, u16(4, 16, 2, 32))
    with pytest.raises(ValueError, match="scales"):
        capi.make_kv_cache(k.astype(np.int8), k.astype(np.int8), np.zeros((4, 16, 2), np.float32), np.zeros((4, 2, 16), np.float32).transpose(0, 2, 1))
    c = capi.make_kv_cache(k, k.copy())
    with pytest.raises(ValueError, match="slots"):
        capi.make_kv_append(c, u16(3, 2, 64), u16(3, 2, 64), np.zeros(3, np.int32))
    with pytest.raises(ValueError, match="k's type"):
        capi.make_kv_append(c, u16(3, 2, 64), u16(3, 4, 64), np.zeros(3, np.int64))
    with pytest.raises(ValueError, match="page_table"):
        capi.make_paged_attention(c, u16(3, 4, 64), u16(3, 4, 64), np.zeros((2, 2), np.int32), np.zeros(3, np.int32))
    with pytest.raises(ValueError, match="out must"):
        capi.make_paged_attention(c, u16(3, 4, 64), u16(3, 4, 32), np.zeros((3, 2), np.int32), np.zeros(3, np.int32))
    with pytest.raises(ValueError, match="ids"):
        capi.make_moe_gate(np.zeros((3, 8), np.float32), 2, np.zeros((3, 4), np.int32))
