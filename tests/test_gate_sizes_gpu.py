"""b200dnn_moe_gate at the largest numbers of experts and tokens at once."""
import pytest
import torch

from serving import run
from test_moe_gate_gpu import capi  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E", [1024, 1021])
def test_as_many_experts_and_tokens_as_a_block_takes(capi, E):  # noqa: F811
    """2048 tokens a block and 1024 experts: what a block keeps is 48 KB and a little more.  Every token's best expert is known."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    T = 2048 * sms - 5
    g = torch.Generator(device="cuda").manual_seed(0)
    best = torch.randint(0, E, (T,), generator=g, device="cuda")
    x = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    x[torch.arange(T, device="cuda"), best] = 1.0
    ids, w = torch.full((T, 1), -7, dtype=torch.int32, device="cuda"), torch.zeros(T, 1, device="cuda")
    counts, rows = torch.full((E,), -7, dtype=torch.int32, device="cuda"), torch.full((T, 1), -7, dtype=torch.int32, device="cuda")
    capi.check(run(capi, capi.lib.b200dnn_moe_gate, capi.make_moe_gate(x, 1, ids, w, renorm=False, expert_counts=counts, slot_to_row=rows)))
    assert torch.equal(ids[:, 0].long(), best)
    e = torch.e
    assert ((w - e / (e + E - 1)).abs() <= 2.0 ** -19 * e / (e + E - 1)).all()
    assert torch.equal(counts.long(), torch.bincount(best, minlength=E))
    want = torch.empty(T, dtype=torch.int64, device="cuda")
    want[best.sort(stable=True)[1]] = torch.arange(T, device="cuda")
    assert torch.equal(rows[:, 0].long(), want)
