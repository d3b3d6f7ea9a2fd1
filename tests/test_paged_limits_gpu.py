"""b200dnn_paged_attention at the ends of its scales and caps: products of zero stay zero, a cap far above the scores changes nothing."""
import pytest
import torch

from test_paged_attention_gpu import capi, check, filled, queries  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,dim", [("bf16", 64), ("s8", 64), ("bf16", 50), ("s8", 40)])
def test_ends(capi, dt, dim):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(dim)
    lens = [100, 17, 0, 300]
    cache, table = filled(g, lens, 2, dim, dt, 16)
    q = queries(g, 4, 4, dim)
    for kw in (dict(softcap=1e36), dict(softcap=1e20), dict(softcap=1e-20), dict(softcap=1e-20, window=9)):
        check(capi, cache, table, lens, q, out="f32", **kw)
    for kw in (dict(scale=1e36), dict(scale=-1e36, softcap=1.0), dict(softcap=1e-36)):
        check(capi, cache, table, lens, torch.zeros_like(q), out="f32", **kw)
