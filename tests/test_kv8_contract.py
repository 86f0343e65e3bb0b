"""What the header promises of the 8-bit cache's calls beside their shapes, without a GPU."""

import pytest

from test_kv8_capi import attn


@pytest.mark.parametrize("nq,nkv,t,d", [(40, 8, 1, 128), (40, 8, 3, 128), (9, 3, 5, 64), (8, 8, 1, 128), (30, 10, 1, 64), (32, 8, 1, 128)])
def test_partials_begin_on_16_bytes(qlib, nq, nkv, t, d):
    """A split's partial of an odd number of rows R takes R (head_dim + 2) + 2 floats."""
    r = t * nq // nkv
    one = 4 * (r * (d + 2) + (2 if r % 2 else 0))
    assert one % 16 == 0
    for splits in (2, 3, 7):
        assert qlib.kv8_attn_workspace(attn(nq=nq, nkv=nkv, t_rows=t, head_dim=d, splits=splits)) == (2 * nkv * splits * one, 0)
