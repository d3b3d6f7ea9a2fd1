"""Serving calls with buffers in host memory inside a stream capture: refused (they are synchronous), and the capture goes on."""
import ctypes as C

import pytest
import torch

from serving import Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from zendnn_b200 import capi as c
    assert c.lib.b200dnn_device_count() > 0, "no CUDA device"
    return c


@pytest.mark.parametrize("pinned", [True, False])
@pytest.mark.parametrize("what", ["slots", "k", "q_out", "table", "lse", "logits", "ids"])
def test_host_buffers_are_not_captured(capi, what, pinned):
    """One buffer of a call in host memory, pinned or not; the call on the device beside it is captured and replayed as if nothing had been asked for."""
    host = lambda t: t.cpu().pin_memory() if pinned else t.cpu()
    at = lambda name, t: host(t) if name == what else t
    cache = Cache(2, 16, 1, 64, "bf16")
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    slots, q_out = torch.arange(3, device="cuda"), torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    good = capi.make_kv_append(cache.desc(capi), k, k, slots, q=k, q_out=q_out)
    if what in ("slots", "k", "q_out"):
        entry = capi.lib.b200dnn_kv_append
        desc = capi.make_kv_append(cache.desc(capi), at("k", k), k, at("slots", slots), q=k, q_out=at("q_out", q_out))
    elif what in ("table", "lse"):
        entry = capi.lib.b200dnn_paged_attention
        desc = capi.make_paged_attention(cache.desc(capi), k, torch.zeros(3, 1, 64, device="cuda"), at("table", torch.zeros(3, 2, dtype=torch.int32, device="cuda")),
                                         torch.ones(3, dtype=torch.int32, device="cuda"), lse=at("lse", torch.zeros(3, 1, device="cuda")))
    else:
        entry = capi.lib.b200dnn_moe_gate
        desc = capi.make_moe_gate(at("logits", torch.zeros(3, 8, device="cuda")), 2, at("ids", torch.zeros(3, 2, dtype=torch.int32, device="cuda")))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        rc = entry(C.byref(desc), st.cuda_stream)
        text = capi.last_error()
        capi.check(capi.lib.b200dnn_kv_append(C.byref(good), st.cuda_stream))
    assert rc == capi.UNIMPLEMENTED and "captured" in text, (rc, text)
    graph.replay()
    torch.cuda.synchronize()
    assert (q_out == 1).all() and (cache.kv[0][0, :3] == 1).all()
