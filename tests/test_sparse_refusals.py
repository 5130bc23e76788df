"""Arguments that attention over drafted trees and over selected pages, page bounds and the selection refuse, through the C ABI (its checks come before any use of the GPU, so the
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


def _bounds(N, geo=None, pool=None, batch=None, **kw):
    a = dict(b=T, step=512)
    a.update(kw)
    geo, pool, batch = geo or _geo(N), pool or _pool(N, v=None), batch or _batch(N)
    return N.lib().ztcp_page_bounds(C.byref(pool), C.byref(batch), C.byref(geo), a["b"], a["step"], None), N.last_error()


def _select(N, geo=None, batch=None, **kw):
    a = dict(q=Q, qs=1024, heads=8, b=T, step=512, pages=8, budget=4, sink=1, recent=1, out=O, work=W, bytes=1 << 30)
    a.update(kw)
    geo, batch = geo or _geo(N), batch or _batch(N)
    rc = N.lib().ztcp_select_pages(a["q"], a["qs"], a["heads"], a["b"], a["step"], a["pages"], C.byref(batch), C.byref(geo),
                                   a["budget"], a["sink"], a["recent"], a["out"], a["work"], a["bytes"], None)
    return rc, N.last_error()


def _selected(N, geo=None, pool=None, batch=None, **kw):
    a = dict(q=Q, qs=1024, out=O, lse=None, heads=8, list=T, listed=4, scale=0.1, work=W, bytes=1 << 30)
    a.update(kw)
    geo, pool, batch = geo or _geo(N), pool or _pool(N), batch or _batch(N)
    rc = N.lib().ztcp_selected_attention(a["q"], a["qs"], a["out"], a["lse"], a["heads"], C.byref(pool), C.byref(batch),
                                         C.byref(geo), a["list"], a["listed"], a["scale"], a["work"], a["bytes"], None)
    return rc, N.last_error()


@pytest.mark.parametrize("kw", [dict(geo=x) for x in BAD_GEO] + [dict(pool=x) for x in BAD_POOL if "v" not in x]
                         + [dict(batch=x) for x in BAD_BATCH])
def test_bounds_and_selected_geometry_pool_and_batch(N, kw):
    made = {k: dict(geo=_geo, pool=_pool, batch=_batch)[k](N, **v) for k, v in kw.items()}
    assert _bounds(N, **made)[0] == N.EINVAL or kw == dict(batch=dict(n_rows=1 << 28))   # (8 query heads to a row are others')
    assert _selected(N, **made)[0] == N.EINVAL
    if "pool" not in made:
        assert _select(N, **made)[0] == N.EINVAL or kw == dict(geo=dict(t=1 << 20, h=1 << 10))   # (no pages are read)


@pytest.mark.parametrize("kw", [dict(b=None), dict(b=T + 8), dict(step=504), dict(step=516)])
def test_bounds_arguments(N, kw):
    rc, why = _bounds(N, **kw)
    assert rc == N.EINVAL and "bounds" in why
    rc, why = _select(N, **kw)
    assert rc == N.EINVAL and "bounds" in why


def test_bounds_overlap_and_width(N):
    assert _bounds(N, b=K + 1024)[0] == N.EOVERLAP
    wide = dict(geo=_geo(N, d=1040, r=0), pool=_pool(N, k_stride=16 * 2 * 1040, v=None))
    assert _bounds(N, **wide, step=4160) == (N.EINVAL, "head_dim must be at most 1024")
    assert _select(N, geo=_geo(N, d=272, r=0), step=2 * 2 * 272) == (N.EINVAL, "head_dim must be at most 256")
    assert _bounds(N, batch=_batch(N, n_seqs=0))[0] == N.OK == _bounds(N, batch=_batch(N, n_rows=0))[0]


@pytest.mark.parametrize("kw", [x for x in BAD_CALL if "scale" not in x and "out" not in x]
                         + [dict(out=None), dict(out=O + 2), dict(pages=0), dict(pages=1 << 31), dict(budget=1), dict(sink=-1),
                            dict(recent=0), dict(sink=4), dict(budget=1 << 31), dict(work=None), dict(work=W + 8), dict(bytes=64)])
def test_select_arguments(N, kw):
    assert _select(N, **kw)[0] == N.EINVAL


def test_select_overlaps_and_workspace(N):
    for kw in (dict(out=Q), dict(out=T + 64), dict(work=Q), dict(work=T), dict(work=O)):
        assert _select(N, **kw)[0] == N.EOVERLAP, kw
    assert _select(N, batch=_batch(N, n_rows=0))[0] == N.OK
    L, bad = N.lib(), C.c_size_t(-1).value
    geo, batch = _geo(N), _batch(N)
    need = L.ztcp_select_pages_workspace(C.byref(batch), 8, C.byref(geo), 8)
    assert 2 * 2 * 4 * 4 <= need < 1 << 20
    assert L.ztcp_select_pages_workspace(C.byref(batch), 0, C.byref(geo), 8) == bad
    assert L.ztcp_select_pages_workspace(C.byref(batch), 8, C.byref(geo), 7) == bad
    for big in (dict(n_rows=(1 << 28) - 1024, max_pages=1 << 26, table_stride=1 << 26), dict(n_rows=1 << 20, max_pages=1 << 26, table_stride=1 << 26)):
        batch = _batch(N, **big)
        assert L.ztcp_select_pages_workspace(C.byref(batch), 8, C.byref(geo), 8) == bad


@pytest.mark.parametrize("kw", BAD_CALL + [dict(list=None), dict(list=T + 2), dict(listed=0), dict(listed=-1), dict(listed=1 << 27)])
def test_selected_arguments(N, kw):
    assert _selected(N, **kw)[0] == N.EINVAL


def test_selected_overlaps(N):
    for kw in (dict(out=T), dict(lse=T + 8), dict(out=Q), dict(out=K + 64), dict(lse=V), dict(lse=O)):
        assert _selected(N, **kw)[0] == N.EOVERLAP, kw
    assert _selected(N, pool=_pool(N, v=None))[0] == N.EINVAL
    assert _selected(N, batch=_batch(N, n_seqs=0))[0] == N.OK


def test_python_checks(N):
    import vlx_tee_amd.attention as A

    x, pages = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    tree = lambda q=x, k=pages, v=pages, m=i32.long()[:, None], **kw: A.tree_attention(q, k, v, i32[None], i32[:1], i32, m, **kw)  # noqa: E731
    for kw, why in ((dict(), "HIP float16 or bfloat16"), (dict(v=None), "single-buffer"), (dict(m=None), "tree_mask must be a tensor"),
                    (dict(q=x.clone().requires_grad_()), "q requires a gradient"), (dict(return_lse=torch.ones(2)), "true or false")):
        with pytest.raises(ValueError, match=why):
            tree(**kw)
    sparse = lambda q=x, k=pages, v=pages, p=i32[:, None, None], **kw: A.selected_attention(q, k, v, i32[None], i32[:1], i32, p, **kw)  # noqa: E731
    for kw, why in ((dict(), "HIP float16 or bfloat16"), (dict(v=None), "single-buffer"), (dict(p=3), "selected must be a tensor"),
                    (dict(k=pages.clone().requires_grad_()), "k_pages requires a gradient"), (dict(return_lse=torch.ones(2)), "true or false")):
        with pytest.raises(ValueError, match=why):
            sparse(**kw)
    b = pages[:, :2]
    with pytest.raises(ValueError, match="HIP float16 or bfloat16"):
        A.page_bounds(pages, b, i32[None], i32[:1], i32)
    for kw, why in ((dict(), "HIP float16 or bfloat16"), (dict(bounds=pages), "n_pages, 2, kv_heads"), (dict(bounds=None), "bounds must be a tensor"),
                    (dict(budget=2.5), "budget must be a whole number"), (dict(q=x.clone().requires_grad_()), "q requires a gradient")):
        a = dict(q=x, bounds=b, page_table=i32[None], kv_lens=i32[:1], q_starts=i32, page_tokens=16, budget=4)
        a.update(kw)
        with pytest.raises(ValueError, match=why):
            A.select_pages(**a)


def test_gradients_and_tangents_are_refused(N):
    """The operators have no derivatives: a tensor that carries one would lose it without a word."""
    import torch.autograd.forward_ad as fwAD
    import vlx_tee_amd.attention as A

    x, pages = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    at, mask, b = (i32[None], i32[:1], i32), i32.long()[:, None], pages[:, :2].clone()
    for name, t, call in (("q", x, lambda t: A.tree_attention(t, pages, pages, *at, mask)),
                          ("v_pages", pages, lambda t: A.tree_attention(x, pages, t, *at, mask)),
                          ("q", x, lambda t: A.selected_attention(t, pages, pages, *at, i32[:, None, None])),
                          ("k_pages", pages, lambda t: A.selected_attention(x, t, pages, *at, i32[:, None, None])),
                          ("q", x, lambda t: A.select_pages(t, b, *at, page_tokens=16, budget=2)),
                          ("bounds", b, lambda t: A.select_pages(x, t, *at, page_tokens=16, budget=2)),
                          ("k_pages", pages, lambda t: A.page_bounds(t, b, *at)), ("bounds", b, lambda t: A.page_bounds(pages, t, *at))):
        with fwAD.dual_level(), torch.no_grad(), pytest.raises(ValueError, match=f"{name} carries a tangent"):
            call(fwAD.make_dual(t, torch.ones_like(t)))
        leaf = t.clone().requires_grad_()
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call(leaf)
        with torch.no_grad(), pytest.raises(ValueError, match="HIP"):
            call(leaf)
