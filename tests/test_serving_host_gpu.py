"""Serving calls with inputs in host memory and outputs on the device: synchronous, as the header says of host buffers."""
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


def busy():
    """Some milliseconds of work in front of the next call on the stream."""
    x = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16)
    for _ in range(30):
        torch.matmul(x, x)


def calls(capi):
    """name -> (entry, descriptor, host array whose contents the call depends on, device output)"""
    pin = lambda t: t.pin_memory()
    cache = Cache(2, 16, 1, 64, "bf16")
    for t in cache.kv:
        t.copy_(torch.arange(2 * 16 * 64, device="cuda").view(2, 16, 1, 64) % 97)
    g = torch.Generator().manual_seed(0)
    k = pin(torch.randn(8, 1, 64, generator=g).to(torch.bfloat16))
    slots = torch.arange(8, device="cuda")
    q, out = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16).cuda(), torch.zeros(2, 2, 64, device="cuda")
    table = pin(torch.tensor([[0, 1], [1, 0]], dtype=torch.int32))
    lens = torch.tensor([20, 17], dtype=torch.int32, device="cuda")
    x, ids = pin(torch.randn(64, 16, generator=g)), torch.zeros(64, 2, dtype=torch.int32, device="cuda")
    return {"kv_append": (capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), k, k, slots), k, cache.kv[0][0, :8]),
            "paged_attention": (capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), q, out, table, lens), table, out),
            "moe_gate": (capi.lib.b200dnn_moe_gate, capi.make_moe_gate(x, 2, ids), x, ids)}


@pytest.mark.parametrize("name", ["kv_append", "paged_attention", "moe_gate"])
def test_a_pinned_input_may_change_behind_the_call(capi, name):
    entry, desc, host, out = calls(capi)[name]
    before = host.clone()
    capi.check(entry(C.byref(desc), stream()))
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    busy()
    capi.check(entry(C.byref(desc), stream()))
    host.zero_()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    host.copy_(before)


def test_an_index_out_of_range_fails_the_call_itself(capi):
    cache = Cache(2, 16, 1, 64, "bf16")
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    assert capi.lib.b200dnn_kv_append(C.byref(capi.make_kv_append(cache.desc(capi), k, k, torch.tensor([0, 50, 1]))), stream()) == capi.FAILURE and "out of range" in capi.last_error()
    out = torch.zeros(1, 1, 64, device="cuda")
    d = capi.make_paged_attention(cache.desc(capi), k[:1], out, torch.tensor([[0, 7]], dtype=torch.int32), torch.tensor([20], dtype=torch.int32, device="cuda"))
    assert capi.lib.b200dnn_paged_attention(C.byref(d), stream()) == capi.FAILURE and "out of range" in capi.last_error()
    capi.check(capi.lib.b200dnn_stream_status(stream()))
