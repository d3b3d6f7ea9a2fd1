"""Captured serving calls replayed on other streams than the one they were captured on: what their kernels report reaches whoever asks there, and no call that has nothing to do with them."""
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


@pytest.mark.parametrize("what", ["slot", "page"])
def test_an_index_out_of_range_is_told_where_the_graph_ran(capi, what):
    cache = Cache(2, 16, 1, 64, "bf16")
    for t in cache.kv:
        t.zero_()
    x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(1, 1, 64, device="cuda")
    slots, table = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    if what == "slot":
        entry, desc, index = capi.lib.b200dnn_kv_append, capi.make_kv_append(cache.desc(capi), x, x, slots), slots
    else:
        entry, desc, index = capi.lib.b200dnn_paged_attention, capi.make_paged_attention(cache.desc(capi), x, out, table, lens), table
    home, away = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=home):
        capi.check(entry(C.byref(desc), home.cuda_stream))
    status = capi.lib.b200dnn_stream_status
    for _ in range(2):
        index.fill_(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(away):
            graph.replay()
        capi.check(status(away.cuda_stream))
        index.fill_(1000)
        torch.cuda.synchronize()
        with torch.cuda.stream(away):
            graph.replay()
        # the capturing stream has not run anything: a call of its own with host buffers is not to blame
        away.synchronize()
        a, got = torch.ones(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8)
        scale = torch.zeros(4)
        capi.check(capi.lib.b200dnn_quant_per_token(a.data_ptr(), capi.DT["bf16"], 4, 64, 64, got.data_ptr(), 64, scale.data_ptr(), capi.DT["f32"], home.cuda_stream))
        assert (got == 127).all()
        assert status(away.cuda_stream) == capi.FAILURE and "out of range" in capi.last_error()
        capi.check(status(away.cuda_stream))
        capi.check(status(home.cuda_stream))
