"""Sizes and parameters at the ends of what the serving entry points take: refused by the checks of the arguments alone, without a GPU."""
import pytest

from test_serving_args import append, attend, capi, gate, refused  # noqa: F401  (fixture)


@pytest.mark.parametrize("T,k,E", [((1 << 31) - 1, 1, 1), ((1 << 31) - 4096, 1, 8), (1 << 27, 16, 64), ((1 << 30) - 2000, 2, 4)])
def test_more_slots_than_places_are_counted_for(capi, T, k, E):  # noqa: F811
    """A block's tokens end below 2^31, the last one's too."""
    d = gate(capi, E=E, k=k)
    d.num_tokens = T
    refused(capi, "b200dnn_moe_gate", d, "too many", capi.UNIMPLEMENTED)
