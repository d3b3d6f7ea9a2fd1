"""b200dnn_moe_layer_routed where a token names one expert several times: bit for bit what it gives with copies of that expert."""
import numpy as np
import pytest
import torch

from serving import stream
from test_serving_host_gpu import capi  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k,S", [(1, 4, 4, 0), (3, 8, 2, 1), (16, 8, 8, 0), (64, 4, 4, 2), (64, 16, 16, 0), (300, 8, 4, 1), (300, 300, 5, 0), (2000, 4, 3, 0)])
@pytest.mark.parametrize("one", [True, False])
def test_one_expert_several_times(capi, T, E, k, S, one):  # noqa: F811
    """Every token the same expert, or each its own; expert e and expert E + e of the wider layer are copies."""
    H, I = 128, 64
    rng = np.random.default_rng(E + T)
    x = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.bfloat16)
    w13, w2 = (torch.from_numpy(rng.integers(-127, 128, (E, *s), dtype=np.int8)).cuda() for s in ((H, 2 * I), (I, H)))
    sh13, sh2 = (torch.from_numpy(rng.integers(-127, 128, (S, *s), dtype=np.int8)).cuda() for s in ((H, 2 * I), (I, H)))
    s13, s2 = torch.full((2 * I,), 1e-3, device="cuda"), torch.full((H,), 1e-3, device="cuda")
    mine = np.repeat(rng.integers(0, E, (1 if one else T, 1)), T if one else 1, 0).astype(np.int32)
    w = torch.rand(T, k, generator=torch.Generator().manual_seed(1)).cuda()
    outs = []
    for copies in (1, k):
        ex = (capi.MoeExpert * (E * copies + S))()
        for e in range(E * copies + S):
            a, b = (w13[e % E], w2[e % E]) if e < E * copies else (sh13[e - E * copies], sh2[e - E * copies])
            ex[e].w13, ex[e].ldb13, ex[e].w13_scale, ex[e].w2, ex[e].ldb2, ex[e].w2_scale = a.data_ptr(), 2 * I, s13.data_ptr(), b.data_ptr(), H, s2.data_ptr()
        ids = torch.from_numpy(mine + E * (np.arange(k, dtype=np.int32) % copies)[None]).cuda().contiguous()
        out = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        capi.check(capi.lib.b200dnn_moe_layer_routed(x.data_ptr(), H, ids.data_ptr(), w.data_ptr(), T, E * copies, S, k, ex, H, I, H, 0, capi.ACT["silu_and_mul"], out.data_ptr(), H, stream()))
        capi.check(capi.lib.b200dnn_stream_status(stream()))
        outs.append(out)
    assert outs[0].abs().sum() > 0 and torch.equal(outs[0], outs[1])
    capi.lib.b200dnn_clear_caches()
