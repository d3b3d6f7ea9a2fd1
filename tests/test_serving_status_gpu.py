"""What the serving calls report, and to whom: an index out of range beside a wait that ran out."""
import ctypes as C

import pytest
import torch

from serving import Cache, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


def append(capi, cache, slots):
    k = torch.ones(len(slots), 1, 64, dtype=torch.bfloat16, device="cuda")
    return capi.make_kv_append(cache.desc(capi), k, k, torch.tensor(slots, device="cuda"))


@pytest.mark.parametrize("bad_first", [False, True])
def test_a_bad_slot_does_not_hide_a_wait_that_ran_out(capi, monkeypatch, bad_first):
    """Both on one stream, in either order: the first check tells of the wait, the next one of the slot."""
    st = stream()
    q, k, v, o = (torch.randn(1, 2, n, 64, device="cuda").bfloat16() for n in (3, 100, 100, 3))
    d = capi.SdpaDesc()
    d.batch, d.num_heads, d.seq_len, d.kv_seq_len, d.head_dim = 1, 2, 3, 100, 64
    for name, x in (("q_stride", q), ("k_stride", k), ("v_stride", v), ("o_stride", o)):
        setattr(d, name, (C.c_int64 * 4)(*x.stride()))
    d.qkv_dt = d.out_dt = capi.DT["bf16"]
    d.query, d.key, d.value, d.output = (x.data_ptr() for x in (q, k, v, o))
    cache = Cache(1, 16, 1, 64, "bf16")
    bad = append(capi, cache, [0, 99])
    monkeypatch.setenv("B200DNN_TEST_NO_LOADS", "1")
    if bad_first:
        capi.check(capi.lib.b200dnn_kv_append(C.byref(bad), st))
    capi.check(capi.lib.b200dnn_sdpa(C.byref(d), st))
    if not bad_first:
        capi.check(capi.lib.b200dnn_kv_append(C.byref(bad), st))
    monkeypatch.delenv("B200DNN_TEST_NO_LOADS")
    assert capi.lib.b200dnn_stream_status(st) == capi.FAILURE and "gave up waiting" in capi.last_error()
    assert capi.lib.b200dnn_stream_status(st) == capi.FAILURE and "out of range" in capi.last_error()
    capi.check(capi.lib.b200dnn_stream_status(st))
    capi.check(capi.lib.b200dnn_sdpa(C.byref(d), st))
    capi.check(capi.lib.b200dnn_stream_status(st))
