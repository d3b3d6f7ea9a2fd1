"""b200dnn_moe_layer_routed on a routing in pinned host memory: the arrays may change behind the call."""
import numpy as np
import pytest
import torch

from serving import stream
from test_serving_host_gpu import busy, capi  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k", [(5, 8, 2), (100, 8, 2), (40, 300, 3)])
@pytest.mark.parametrize("what", ["ids", "weights"])
def test_a_routing_in_pinned_memory(capi, what, T, E, k):  # noqa: F811
    H, I = 128, 64
    rng = np.random.default_rng(E)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
    w13, w2 = (torch.from_numpy(rng.integers(-127, 128, (E, *s), dtype=np.int8)).cuda() for s in ((H, 2 * I), (I, H)))
    s13, s2 = torch.full((2 * I,), 1e-3, device="cuda"), torch.full((H,), 1e-3, device="cuda")
    ex = (capi.MoeExpert * E)()
    for e in range(E):
        ex[e].w13, ex[e].ldb13, ex[e].w13_scale, ex[e].w2, ex[e].ldb2, ex[e].w2_scale = w13[e].data_ptr(), 2 * I, s13.data_ptr(), w2[e].data_ptr(), H, s2.data_ptr()
    ids = torch.from_numpy(np.stack([rng.choice(E - 1, k, replace=False) + 1 for _ in range(T)]).astype(np.int32))
    arrays = {"ids": ids, "weights": torch.rand(T, k, generator=torch.Generator().manual_seed(1))}
    arrays = {n: t.pin_memory() if n == what else t.cuda() for n, t in arrays.items()}
    out = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")

    def call():
        capi.check(capi.lib.b200dnn_moe_layer_routed(x.data_ptr(), H, arrays["ids"].data_ptr(), arrays["weights"].data_ptr(), T, E, 0, k, ex, H, I, H, 0, capi.ACT["silu_and_mul"],
                                                     out.data_ptr(), H, stream()))

    call()
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    busy()
    call()
    arrays[what].zero_()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    capi.lib.b200dnn_clear_caches()
