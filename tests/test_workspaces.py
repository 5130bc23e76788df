"""What the operators on hot pages keep between their kernels does not grow with the call beyond a gigabyte (and what grows with
the batch's tables alone): larger calls are done in parts."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import sparse_reference as R
from test_gpu_sparse import BF, FP, _select_case
from test_hot_refusals import N, _batch, _geo, _pool  # noqa: F401  (N: the module's fixture)

MOST = 1 << 30


@pytest.mark.parametrize("rows,pages,kv,group", [(65536, 4096, 8, 4), (65536, 8192, 8, 8), (100000, 500, 1, 1), (3, 1 << 20, 8, 4), (1, 1 << 22, 64, 1)])
def test_selection(N, rows, pages, kv, group):
    batch, geo = _batch(N, n_rows=rows, max_pages=pages, table_stride=pages, n_seqs=4), _geo(N, h=kv)
    need = N.lib().ztcp_select_pages_workspace(C.byref(batch), 1 << 20, C.byref(geo), kv * group)
    row = 4 * kv * pages * (2 if pages > 12288 else 1)   # scores, and keys where these are not in local memory
    assert row <= need <= max(MOST, row) + 4 * (4 * kv * (-(-pages // 16)) + 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group,d", [(BF, 2, 16), (FP, 9, 16), (BF, 4, 96), (FP, 1, 256)])
def test_selection_in_parts(hip, dtype, group, d):
    """Tables of 8,192 columns and 39,855 rows: three parts of 13,285 rows, with sequences across both borders.  Most rows see
    no page, which costs the reference nothing."""
    import vlx_tee_amd.attention as A

    lens = [(13270, 0), (40, 1200), (13090, 0), (300, 400), (13154, 0), (1, 1200)]
    print("case", dtype, group, d, flush=True)
    c = _select_case(lens, 2, group, d, 1, dtype, seed=d, missing=0.1)
    wide = torch.full((len(lens), 8192), -1, dtype=torch.int32, device="cuda")
    wide[:, :c["table"].shape[1]] = c["table"]
    out = torch.full((c["q"].shape[0], 2, 9), -7, dtype=torch.int32, device="cuda")
    want = R.select(c["q"], c["b"], wide, c["lens"], c["starts"], 1, 9, 1, 2, out)
    got = A.select_pages(c["q"], c["b"], wide, c["lens"], c["starts"], page_tokens=1, budget=9, sink=1, recent=2, out=out)
    assert torch.equal(got.cpu(), want), int((got.cpu() != want).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kv,group,d", [(16384, 8, 4, 128), (65536, 8, 8, 256), (8192, 32, 1, 64), (40, 1, 8, 128)])
def test_pieces_of_trees(hip, N, rows, kv, group, d):
    for pages in (3, 300, 9000):
        batch, geo = _batch(N, n_rows=rows, max_pages=pages, table_stride=pages, n_seqs=4), _geo(N, h=kv, d=d)
        pool = _pool(N, k_stride=16 * kv * d, v_stride=16 * kv * d)
        need = N.lib().ztcp_tree_attention_workspace(C.byref(batch), C.byref(pool), C.byref(geo), kv * group)
        assert need <= MOST + 16, (pages, need)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,group,d", [(8400, 4, 128), (2600, 25, 64)])
def test_trees_among_many_rows(hip, rows, group, d):
    """Of arrays for many rows, whose pieces' results would pass a gigabyte: most rows are no sequence's."""
    import vlx_tee_amd.attention as A
    from test_gpu_tree import _case, _close

    print("case", rows, group, d, flush=True)
    c = _case([(40, 1700), (64, 2500), (3, 900)], 8, group, d, 16, BF, words=2)
    real = c["q"].shape[0]
    q = torch.zeros((rows, *c["q"].shape[1:]), dtype=BF, device="cuda")
    mask = torch.zeros((rows, c["mask"].shape[1]), dtype=torch.int64, device="cuda")
    q[:real], mask[:real] = c["q"], c["mask"]
    out = torch.full_like(q, 7.0)
    got, lse = A.tree_attention(q, c["k"], c["v"], c["table"], c["lens"], c["starts"], mask, return_lse=True, out=out)
    want = R.tree(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["mask"], d ** -0.5)
    _close(got[:real], want[0], want[2], "out")
    _close(lse[:real], want[1], want[3], "lse")
    assert bool((got[real:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,kv,group,listed,pages", [(65536, 32, 1, 128, 8192), (65536, 8, 4, 128, 8192), (1 << 18, 8, 8, 512, 1 << 17)])
def test_lists_of_blocks(hip, N, rows, kv, group, listed, pages):
    batch, geo = _batch(N, n_rows=rows, max_pages=pages, table_stride=pages, n_seqs=4), _geo(N, h=kv)
    pool = _pool(N, k_stride=16 * kv * 128, v_stride=16 * kv * 128)
    need = N.lib().ztcp_selected_attention_workspace(C.byref(batch), C.byref(pool), C.byref(geo), kv * group, listed)
    assert MOST // 4 < need <= MOST + 256, need


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t", [(BF, 16), (FP, 13)])
def test_lists_in_parts(hip, dtype, t):
    """92,560 rows over tables of 8,192 columns: lists of 196 KiB a workgroup, two launches of 2,900 workgroups of 8 heads.
    The sequences between those that are looked at have no tokens."""
    import vlx_tee_amd.attention as A
    from test_gpu_sparse import _attend_case, _close

    print("case", dtype, t, flush=True)
    c = _attend_case([(300, 700), (260, 500)], 8, 1, 32, t, dtype, 64, seed=4)
    lens = [(46000, 0), (300, 700), (46000, 0), (260, 500)]
    table = torch.full((4, 8192), -1, dtype=torch.int32, device="cuda")
    table[1::2, :c["table"].shape[1]] = c["table"]
    starts = torch.tensor([0] + [n for n, _ in lens], device="cuda").cumsum(0).int()
    rows = int(starts[-1])
    at = torch.cat([torch.arange(46000, 46300), torch.arange(92300, 92560)]).cuda()
    q = torch.zeros((rows, *c["q"].shape[1:]), dtype=dtype, device="cuda")
    picked = torch.full((rows, *c["picked"].shape[1:]), -1, dtype=torch.int32, device="cuda")
    q[at], picked[at] = c["q"], c["picked"]
    kv_lens = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
    out, lse = A.selected_attention(q, c["k"], c["v"], table, kv_lens, starts, picked, return_lse=True)
    c["table"] = table[1::2]   # (which columns there are tells what a list's entry is)
    want = R.selected(*(c[x] for x in ("q", "k", "v", "table", "lens", "starts", "picked")), 32 ** -0.5)
    _close(out[at], want[0], want[2], "out")
    _close(lse[at], want[1], want[3], "lse")
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((out[rest] == 0).all()) and bool((lse[rest] == -float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lens,group", [([(300, 700), (260, 500)], 4), ([(1, 900), (2, 300)], 4)])
@pytest.mark.parametrize("off", [0, 16, 48, 112])
def test_a_workspace_anywhere(hip, N, lens, group, off):
    """Any 16-byte aligned workspace of the size that is asked for: lists lie in lines of their own within it, and nothing
    around it is written."""
    import vlx_tee_amd.attention as A
    from test_gpu_sparse import _attend_case

    print("case", lens, off, flush=True)
    c = _attend_case(lens, 8, group, 64, 16, BF, 40, seed=2)
    q, k, v, table = c["q"].contiguous(), c["k"], c["v"], c["table"]
    want = A.selected_attention(q, k, v, table, c["lens"], c["starts"], c["picked"], return_lse=True)
    rows, heads, d = q.shape
    geo = N.geometry(16, 8, d, 0, 1, False)
    step = k.stride(0)
    pool = N.PagePool(k=k.data_ptr(), v=v.data_ptr(), n_pages=k.shape[0], k_stride=step, v_stride=step)
    batch = N.PagedBatch(page_table=table.data_ptr(), table_stride=table.stride(0), max_pages=table.shape[1],
                         kv_lens=c["lens"].data_ptr(), q_starts=c["starts"].data_ptr(), n_seqs=len(lens), n_rows=rows, max_q_len=0)
    L = N.lib()
    need = L.ztcp_selected_attention_workspace(C.byref(batch), C.byref(pool), C.byref(geo), heads, 40)
    room = torch.full((need + 512,), 0x5A, dtype=torch.uint8, device="cuda")
    base = -room.data_ptr() % 128 + off
    out, lse = torch.empty_like(q), torch.empty((rows, heads), device="cuda")
    for size, rc in ((need - 1, N.EINVAL), (need, N.OK)):
        if need:
            assert L.ztcp_selected_attention(q.data_ptr(), heads * d, out.data_ptr(), lse.data_ptr(), heads, C.byref(pool), C.byref(batch),
                                             C.byref(geo), c["picked"].data_ptr(), 40, d ** -0.5, room.data_ptr() + base, size,
                                             torch.cuda.current_stream().cuda_stream) == rc
    assert need and torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert bool((room[:base] == 0x5A).all()) and bool((room[base + need:] == 0x5A).all())
    if lens[0][0] > 1:   # blocks
        assert bool((room[base:base + -(room.data_ptr() + base) % 128] == 0x5A).all())
