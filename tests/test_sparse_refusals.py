"""Arguments that attention over drafted trees refuses, through the C ABI (its checks come before any use of the GPU, so the
addresses here are never read) and the Python module.  No GPU needed."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from test_hot_refusals import BAD_GEO, BAD_POOL, K, N, O, Q, V, W, _batch, _geo, _pool  # noqa: F401  (N: the module's fixture)

INF, NAN, T = float("inf"), float("nan"), 0x60000000
BAD_BATCH = [dict(n_seqs=-1), dict(n_seqs=1 << 24), dict(n_rows=-1), dict(n_rows=1 << 31), dict(max_q_len=-1), dict(max_pages=0),
             dict(max_pages=1 << 28), dict(page_table=None), dict(kv_lens=None), dict(q_starts=None), dict(table_stride=3),
             dict(n_rows=1 << 28)]
BAD_CALL = [dict(heads=0), dict(heads=7), dict(heads=1 << 17), dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF),
            dict(q=None), dict(q=Q + 8), dict(qs=1020), dict(qs=512), dict(out=None), dict(out=O + 4)]


def _tree(N, geo=None, pool=None, batch=None, **kw):
    a = dict(q=Q, qs=1024, out=O, lse=None, heads=8, mask=T, words=1, scale=0.1, work=W, bytes=1 << 30)
    a.update(kw)
    geo, pool, batch = geo or _geo(N), pool or _pool(N), batch or _batch(N)
    rc = N.lib().ztcp_tree_attention(a["q"], a["qs"], a["out"], a["lse"], a["heads"], C.byref(pool), C.byref(batch),
                                     C.byref(geo), a["mask"], a["words"], a["scale"], a["work"], a["bytes"], None)
    return rc, N.last_error()


@pytest.mark.parametrize("kw", [dict(geo=x) for x in BAD_GEO] + [dict(pool=x) for x in BAD_POOL] + [dict(batch=x) for x in BAD_BATCH])
def test_tree_geometry_pool_and_batch(N, kw):
    made = {k: dict(geo=_geo, pool=_pool, batch=_batch)[k](N, **v) for k, v in kw.items()}
    assert _tree(N, **made)[0] == N.EINVAL


@pytest.mark.parametrize("kw", BAD_CALL + [dict(mask=None), dict(mask=T + 4), dict(words=0), dict(words=-1), dict(words=1 << 26)])
def test_tree_arguments(N, kw):
    assert _tree(N, **kw)[0] == N.EINVAL


def test_tree_needs_both_buffers_and_a_pool_of_narrow_heads(N):
    assert _tree(N, pool=_pool(N, v=None))[0] == N.EINVAL
    wide = dict(geo=_geo(N, d=272, r=0), pool=_pool(N, k_stride=16 * 2 * 272, v_stride=16 * 2 * 272))
    assert _tree(N, **wide) == (N.EINVAL, "head_dim must be at most 256")


def test_tree_overlaps(N):
    for kw in (dict(out=T), dict(lse=T + 8), dict(out=Q), dict(out=K + 64), dict(lse=V), dict(lse=O)):
        assert _tree(N, **kw)[0] == N.EOVERLAP, kw
    assert _tree(N, batch=_batch(N, n_seqs=0))[0] == N.OK == _tree(N, batch=_batch(N, n_rows=0))[0]


def test_python_checks(N):
    import vlx_tee_amd.attention as A

    x, pages = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    tree = lambda q=x, k=pages, v=pages, m=i32.long()[:, None], **kw: A.tree_attention(q, k, v, i32[None], i32[:1], i32, m, **kw)  # noqa: E731
    for kw, why in ((dict(), "HIP float16 or bfloat16"), (dict(v=None), "single-buffer"), (dict(m=None), "tree_mask must be a tensor"),
                    (dict(q=x.clone().requires_grad_()), "q requires a gradient"), (dict(return_lse=torch.ones(2)), "true or false")):
        with pytest.raises(ValueError, match=why):
            tree(**kw)
