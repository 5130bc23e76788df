"""Sizes at the ends of what the operators on hot pages take, through the C ABI (its checks come before any use of the
GPU, so the addresses are never read).  No GPU needed."""
from __future__ import annotations

import ctypes as C

import pytest

from test_hot_refusals import N, _attend, _batch, _geo, _mass, _pool  # noqa: F401  (N: the module's fixture)


def _one_head(N):
    return dict(geo=_geo(N, h=1), pool=_pool(N, k_stride=2048, v_stride=2048))


@pytest.mark.parametrize("rows", [(1 << 31) - 1, (1 << 31) - 1023])
def test_rows_whose_blocks_pass_2_31_are_refused(N, rows):
    """Kernels count rows in blocks of up to 128, and the next block's first row has to be a 32-bit number too."""
    batch = _batch(N, n_rows=rows)
    for call, kw in ((_attend, dict(bytes=1 << 62)), (_mass, {})):
        rc, why = call(N, **_one_head(N), batch=batch, heads=1, qs=128, **kw)
        assert rc == N.EINVAL and "n_rows * q_heads" in why, (rc, why)
    one = _one_head(N)
    assert N.lib().ztcp_paged_attention_workspace(C.byref(batch), C.byref(one["pool"]), C.byref(one["geo"]), 1) == \
        C.c_size_t(-1).value
    assert "n_rows * q_heads" in N.last_error()
