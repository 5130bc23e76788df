"""GPU tests of attention for drafted tokens that form a tree, against its formula in 64 bits (tests/sparse_reference.py,
which derives the bounds)."""
from __future__ import annotations

import math

import pytest
import torch

import sparse_reference as R

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def A(hip):
    import vlx_tee_amd.attention as A

    return A


def _say(*what):
    print("case", *what, flush=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(got, want, tol, what):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    ok = torch.isnan(want) | (got == want) | ((got - want).abs() <= tol)
    assert bool(ok.all()), (what, float((got - want).abs().nan_to_num(0, 0, 0).max()), int((~ok).sum()))


def random_masks(counts, words, gen, kind="tree"):
    """A tree's lines of ancestors, or any bits."""
    n = sum(counts)
    if kind == "any":
        return torch.randint(-2 ** 63, 2 ** 63 - 1, (n, words), generator=gen)
    out, at = torch.zeros((n, words), dtype=torch.int64), 0
    for c in counts:
        for i in range(c):
            parent = int(torch.randint(max(-1, i - 5), i, (1,), generator=gen)) if i else -1
            if parent >= 0:
                out[at + i] = out[at + parent]
            if i // 64 < words:
                out[at + i, i // 64] |= -2 ** 63 if i % 64 == 63 else 1 << (i % 64)
        at += c
    return out


def _case(lens, kv, group, d, t, dtype, *, words=None, kind="tree", seed=0, missing=0.0, strided=False):
    """lens: [(new tokens, tokens)]"""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-x // t) for _, x in lens]
    mp, n_pages = max(max(need), 1), sum(need) + 2
    ids, table, at = torch.randperm(n_pages, generator=gen).int(), torch.full((len(lens), mp), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    if missing:
        table[torch.rand(table.shape, generator=gen) < missing] = n_pages + 3
    counts = [q for q, _ in lens]
    rows = sum(counts)
    mask = random_masks(counts, words or max(1, -(-max(counts) // 64)), gen, kind)
    heads = kv * group
    q = torch.randn((rows, heads + (3 if strided else 0), d), generator=gen).to(dtype).cuda()[:, :heads]
    pages = [torch.randn((n_pages, t, kv, d), generator=gen).to(dtype).cuda() for _ in range(2)]
    return dict(q=q, k=pages[0], v=pages[1], table=table.cuda(), lens=_i32([x for _, x in lens]),
                starts=_i32([0] + torch.tensor(counts).cumsum(0).tolist()), mask=mask.cuda())


def _run(A, c, **kw):
    return A.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["mask"], return_lse=True, **kw)


def _check(A, c, what, **kw):
    out, lse = _run(A, c, **kw)
    want = R.tree(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["mask"], kw.get("scale", c["q"].shape[2] ** -0.5))
    _close(out, want[0], want[2], (what, "out"))
    _close(lse, want[1], want[3], (what, "lse"))
    return out, lse


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,group,d,t", [
    ([(1, 1)], 1, 1, 64, 16), ([(5, 5)], 2, 2, 128, 16), ([(37, 301)], 5, 3, 96, 13), ([(8, 40), (3, 900), (0, 33), (16, 16)], 2, 4, 128, 16),
    ([(64, 700), (24, 130), (63, 64)], 2, 4, 128, 16), ([(130, 400), (65, 65)], 1, 2, 64, 64), ([(20, 517)], 2, 1, 256, 7),
    ([(33, 260), (2, 1999)], 1, 8, 80, 1), ([(100, 2500), (4, 30)], 1, 6, 192, 100), ([(12, 1500)], 2, 4, 112, 32),
    ([(200, 1300)], 1, 1, 16, 16), ([(7, 2100)] * 9, 1, 2, 128, 64)])
def test_tree(A, lens, kv, group, d, t, dtype):
    _say("tree", lens, kv, group, d, t, dtype)
    for seed, (kind, missing, hint) in enumerate([("tree", 0.0, None), ("any", 0.0, max(q for q, _ in lens)), ("tree", 0.15, 1)]):
        c = _case(lens, kv, group, d, t, dtype, kind=kind, seed=seed, missing=missing, strided=seed == 1)
        _check(A, c, (lens, d, seed), max_q_len=hint)


def test_a_line_is_paged_attention(A):
    """A tree without branches is a chunk: the results are those of paged_attention.  The two may cut the tokens into other
    pieces, so each may be off by the formula's bound."""
    _say("tree as a line")
    for lens in ([(6, 500), (3, 20)], [(70, 900), (12, 12)]):
        c = _case(lens, 2, 4, 128, 16, BF)
        for s, (n, _) in enumerate(lens):
            for i in range(n):
                row = (1 << (i + 1)) - 1
                words = [(row >> (64 * w)) & (2 ** 64 - 1) for w in range(c["mask"].shape[1])]
                c["mask"][int(c["starts"][s]) + i] = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in words])
        out, lse = _run(A, c)
        want = A.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], return_lse=True)
        _, _, out_tol, lse_tol = R.tree(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["mask"], 128 ** -0.5)
        _close(out, want[0].cpu().double(), 2 * out_tol, ("line", "out"))
        _close(lse, want[1].cpu().double(), 2 * lse_tol, ("line", "lse"))


def test_masks_that_leave_nothing(A):
    """Rows that see no token: zeros and -inf; bits of tokens that are not there; too few words."""
    _say("tree, empty masks")
    for lens, words in (([(9, 9), (5, 40)], 1), ([(40, 40), (90, 120)], 1), ([(3, 3)], 5)):
        c = _case(lens, 2, 2, 64, 16, BF, words=words, kind="any", seed=3)
        c["mask"][1], c["mask"][2] = 0, -1
        out, lse = _check(A, c, ("empty", lens))
        assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


def test_numbers_that_a_row_does_not_see(A):
    """NaN and infinities of K and V in drafted tokens reach the rows that see them and no others, those behind the
    sequence nobody; also in the context, which every row sees."""
    _say("tree, NaN and infinities")
    for lens in ([(9, 100), (3, 50)], [(70, 200), (30, 30)]):
        for where in ("draft", "context"):
            c = _case(lens, 2, 2, 64, 16, BF, seed=4)
            n, total = lens[0]
            for j, (pool, value) in zip((1, 4, 6), ((c["v"], math.nan), (c["v"], math.inf), (c["k"], math.nan))):
                place = total - n + j if where == "draft" else 8 * j
                pool[int(c["table"][0, place // 16]), place % 16, 1] = value
            for s, (_, total) in enumerate(lens):   # behind the end
                if total % 16:
                    c["v"][int(c["table"][s, total // 16]), total % 16:] = math.nan
                    c["k"][int(c["table"][s, total // 16]), total % 16:] = math.inf
            out, lse = _run(A, c)
            want = R.tree(*(c[x] for x in ("q", "k", "v", "table", "lens", "starts", "mask")), 64 ** -0.5)
            bad = torch.isnan(want[1])
            assert torch.equal(torch.isnan(lse.cpu()), bad)
            for g, w, tol in ((out, want[0], want[2]), (lse, want[1], want[3])):
                g = g.cpu().double()
                keep = ~bad[..., None].expand_as(w) if w.dim() == 3 else ~bad
                same = (g == w) | (torch.isnan(g) & torch.isnan(w)) | ((g - w).abs() <= tol)
                assert bool(same[keep].all()), (lens, where)


def test_wrong_starts_and_lengths_stay_inside(A):
    """Rows of no sequence keep what out holds; lengths shorter than the new tokens, starts beyond the rows."""
    _say("tree, wrong starts")
    c = _case([(6, 60), (10, 200)], 2, 4, 128, 16, BF, seed=6)
    c["lens"], c["starts"] = _i32([3, 10 ** 6]), _i32([2, 7, 99])
    for rows_hint in (None, 1):
        out = torch.full_like(c["q"], 7.0).contiguous()
        got, lse = _run(A, c, out=out, max_q_len=rows_hint)
        want = R.tree(*(c[x] for x in ("q", "k", "v", "table", "lens", "starts", "mask")), 128 ** -0.5)
        assert bool((got[:2] == 7).all())
        _close(got[2:], want[0][2:], want[2][2:], "wrong starts")


def test_same_results_captured_and_on_another_stream(A):
    _say("tree, graph and stream")
    c = _case([(24, 900), (3, 77), (60, 400)], 2, 4, 128, 16, BF, seed=8)
    want = _run(A, c)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = _run(A, c)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(A, c)
    for turn in range(3):
        c["q"].copy_(torch.randn(c["q"].shape, device="cuda"))
        eager = _run(A, c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1]), turn
