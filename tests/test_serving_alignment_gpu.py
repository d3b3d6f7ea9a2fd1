"""Addresses that are no multiple of their elements' size: refused before any launch."""
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


def descriptors(capi):
    cache, wide = Cache(2, 16, 1, 64, "s8"), Cache(2, 16, 1, 64, "bf16")
    k, slots, at = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda"), torch.arange(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    tab = torch.ones(4, 32, device="cuda")
    table, lens, rows = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 1, device="cuda")
    two = lambda: torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    return {"append": (capi.lib.b200dnn_kv_append, lambda: capi.make_kv_append(cache.desc(capi), k, k, slots, q=k, q_out=torch.zeros_like(k), positions=at, cos=tab, sin=tab)),
            "append bf16": (capi.lib.b200dnn_kv_append, lambda: capi.make_kv_append(wide.desc(capi), k.float(), k.float(), slots)),
            "attend": (capi.lib.b200dnn_paged_attention, lambda: capi.make_paged_attention(cache.desc(capi), k, torch.zeros(3, 1, 64, device="cuda"), table, lens, sinks=rows[0], lse=rows)),
            "attend bf16": (capi.lib.b200dnn_paged_attention, lambda: capi.make_paged_attention(wide.desc(capi), k, torch.zeros_like(k), table, lens)),
            "gate": (capi.lib.b200dnn_moe_gate, lambda: capi.make_moe_gate(torch.zeros(3, 8, device="cuda"), 2, two(), torch.zeros(3, 2, device="cuda"), bias=torch.zeros(8, device="cuda"),
                                                                           expert_counts=torch.zeros(8, dtype=torch.int32, device="cuda"), slot_to_row=two()))}


@pytest.mark.parametrize("vouched", [True, False])
@pytest.mark.parametrize("name,fields", [
    ("append", [("k", 1), ("v", 1), ("q", 1), ("q_out", 1), ("slots", 4), ("positions", 2), ("cos_table", 2), ("sin_table", 1), ("cache.key_scale", 2), ("cache.value_scale", 1)]),
    ("append bf16", [("k", 2), ("v", 1), ("cache.key", 1), ("cache.value", 1)]),
    ("attend", [("q", 1), ("out", 2), ("page_table", 2), ("seq_lens", 1), ("sinks", 2), ("lse", 1), ("cache.key_scale", 2)]),
    ("attend bf16", [("out", 1), ("cache.key", 1), ("cache.value", 1)]),
    ("gate", [("logits", 2), ("bias", 1), ("ids", 2), ("weights", 2), ("expert_counts", 1), ("slot_to_row", 2)])])
def test_addresses_between_elements(capi, name, fields, vouched):
    entry, make = descriptors(capi)[name]
    for field, off in fields:
        d = make()
        if not vouched:
            d.device = 0
        capi.check(entry(C.byref(d), stream()))
        part = d.cache if field.startswith("cache.") else d
        field = field.split(".")[-1]
        setattr(part, field, getattr(part, field) + off)
        assert entry(C.byref(d), stream()) == capi.FAILURE and "multiple" in capi.last_error(), (field, capi.last_error())
    capi.check(capi.lib.b200dnn_stream_status(stream()))
