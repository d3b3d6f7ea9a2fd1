"""Sizes and parameters at the ends of what the serving entry points take: refused by the checks of the arguments alone, without a GPU."""
import pytest

from test_serving_args import append, attend, capi, gate, refused  # noqa: F401  (fixture)


@pytest.mark.parametrize("T,k,E", [((1 << 31) - 1, 1, 1), ((1 << 31) - 4096, 1, 8), (1 << 27, 16, 64), ((1 << 30) - 2000, 2, 4)])
def test_more_slots_than_places_are_counted_for(capi, T, k, E):  # noqa: F811
    """A block's tokens end below 2^31, the last one's too."""
    d = gate(capi, E=E, k=k)
    d.num_tokens = T
    refused(capi, "b200dnn_moe_gate", d, "too many", capi.UNIMPLEMENTED)


@pytest.mark.parametrize("scale", [1e300, -1e39, 1e38, -2.0 ** 121])
def test_scales_that_leave_32_bits(capi, scale):  # noqa: F811
    """The scale, times what the kernel folds into it, is a finite f32."""
    d = attend(capi)
    d.scale = scale
    refused(capi, "b200dnn_paged_attention", d, "scale", capi.UNIMPLEMENTED)


@pytest.mark.parametrize("softcap", [1e-40, 1e-39, 2e36, 3e38])
def test_caps_that_leave_32_bits(capi, softcap):  # noqa: F811
    """scale / softcap and softcap log2(e) are finite f32, and no denormal loses bits."""
    d = attend(capi)
    d.softcap = softcap
    refused(capi, "b200dnn_paged_attention", d, "softcap", capi.UNIMPLEMENTED)


def test_caps_and_scales_within_32_bits_are_taken(capi):  # noqa: F811
    """Up to the look at the sequences' number, of which there is none."""
    import ctypes as C
    for scale, softcap in ((0.0, 1e-36), (0.0, 1e36), (1e36, 1.0), (-1e-300, 30.0), (1e-44, 0.0), (1e36, 0.0)):
        d = attend(capi)
        d.scale, d.softcap, d.num_seqs = scale, softcap, 0
        assert capi.lib.b200dnn_paged_attention(C.byref(d), None) == capi.SUCCESS, capi.last_error()


def test_more_rows_than_a_grid_has(capi):  # noqa: F811
    """Eight rows a block, and fewer than 2^31 blocks."""
    d = append(capi)
    for T, heads in ((1717986918, 6), (1561806289, 7), (572662306, 26), ((1 << 31) - 1, 5)):
        d.num_tokens, d.q_heads = T, heads
        assert (T * (heads + 4) + 7) // 8 >= 1 << 31
        refused(capi, "b200dnn_kv_append", d, "too many", capi.UNIMPLEMENTED)
