"""What the Python helpers of the serving calls refuse beside the checks of test_serving_args.py."""
import numpy as np
import pytest

from test_serving_args import cache, capi, u16  # noqa: F401  (fixture)


def test_tables_without_positions(capi):  # noqa: F811
    """Rows that are to be rotated by tables have a position."""
    c, k, slots, tab = cache(capi), u16(3, 2, 64), np.zeros(3, np.int64), np.zeros((8, 32), np.float32)
    for kw in (dict(cos=tab, sin=tab), dict(cos=tab), dict(sin=tab)):
        with pytest.raises(ValueError, match="positions"):
            capi.make_kv_append(c, k, k, slots, **kw)
    assert capi.make_kv_append(c, k, k, slots).rotary_dim == 0
    assert capi.make_kv_append(c, k, k, slots, positions=np.zeros(3, np.int32), cos=tab, sin=tab).rotary_dim == 64
