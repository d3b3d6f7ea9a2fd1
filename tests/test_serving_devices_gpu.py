"""Serving calls whose buffers lie on several devices: refused, whichever buffer it is."""
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


@pytest.mark.parametrize("what", ["k", "slots", "q_out", "table", "out", "logits", "ids"])
def test_a_buffer_of_another_device(capi, what):
    """(A call looks at its pointers before it launches anything.)"""
    if torch.cuda.device_count() < 2:
        pytest.skip("two devices")
    at = lambda name, t: t.to("cuda:1") if name == what else t
    cache = Cache(2, 16, 1, 64, "bf16")
    k, slots = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda"), torch.arange(3, device="cuda")
    if what in ("k", "slots", "q_out"):
        entry, d = capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), at("k", k), k, at("slots", slots), q=k, q_out=at("q_out", torch.zeros_like(k)))
    elif what in ("table", "out"):
        entry, d = capi.lib.b200dnn_paged_attention, capi.make_paged_attention(
            cache.desc(capi), k, at("out", torch.zeros_like(k)), at("table", torch.zeros(3, 2, dtype=torch.int32, device="cuda")), torch.ones(3, dtype=torch.int32, device="cuda"))
    else:
        entry, d = capi.lib.b200dnn_moe_gate, capi.make_moe_gate(at("logits", torch.zeros(3, 8, device="cuda")), 2, at("ids", torch.zeros(3, 2, dtype=torch.int32, device="cuda")))
    assert d.device == 0
    assert entry(C.byref(d), stream()) == capi.FAILURE and "lies on device 1" in capi.last_error()
