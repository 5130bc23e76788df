"""GPU tests of page bounds, the selection of pages and attention over selected pages, against their formulas in 64 bits
(tests/sparse_reference.py, which derives the bounds).  Bounds are numbers of the keys and selections whole numbers: both have
to be equal."""
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


def _batch(lens, t, gen, missing=0.0, shared=2):
    """lens: [(new tokens, tokens)] -> table, lengths, starts, pages of the pool"""
    need = [-(-x // t) for _, x in lens]
    mp, n_pages = max(max(need), 1), sum(need) + shared
    ids, table, at = torch.randperm(n_pages, generator=gen).int(), torch.full((len(lens), mp), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    if missing:
        table[torch.rand(table.shape, generator=gen) < missing] = n_pages + 3
    return table.cuda(), _i32([x for _, x in lens]), _i32([0] + torch.tensor([q for q, _ in lens]).cumsum(0).tolist()), n_pages


def _same(got, want, what):
    got, want = got.cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7, 5, -5), want.nan_to_num(7, 5, -5)), what


# ---- bounds ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,d,t", [
    ([(1, 1)], 1, 16, 16), ([(1, 700), (1, 16), (1, 17)], 8, 128, 16), ([(300, 300), (0, 50), (37, 999)], 5, 96, 13),
    ([(64, 1000), (5, 5)], 2, 64, 1), ([(900, 2000)], 3, 256, 100), ([(3, 500)] * 70, 1, 80, 7), ([(20, 400)], 1, 576, 64),
    ([(7000, 9000), (1, 3)], 2, 64, 16), ([(40, 5000)], 2, 112, 3000)])
def test_bounds(A, lens, kv, d, t, dtype):
    _say("bounds", lens[:3], kv, d, t, dtype)
    for seed, (hint, missing) in enumerate([(None, 0.0), (max(q for q, _ in lens), 0.1), (1, 0.0)]):
        gen = torch.Generator().manual_seed(seed)
        table, length, starts, n_pages = _batch(lens, t, gen, missing)
        k = torch.randn((n_pages, t, kv, d), generator=gen).to(dtype).cuda()
        before = torch.full((n_pages, 2, kv, d), 9.0, dtype=dtype, device="cuda")
        want = R.bounds(k, before, table, length, starts)
        got = A.page_bounds(k, before, table, length, starts, max_q_len=hint)
        assert got.data_ptr() == before.data_ptr()
        _same(got, want, (lens[:3], seed))


def test_bounds_of_odd_numbers(A):
    """NaN of either sign and infinities among the keys; NaN behind the sequence's end; pools with padding."""
    _say("bounds, odd numbers")
    for dtype in (BF, FP):
        gen = torch.Generator().manual_seed(1)
        table, length, starts, n_pages = _batch([(40, 90), (3, 20)], 16, gen)
        pool = torch.randn((n_pages, 3, 16, 2, 64), generator=gen).to(dtype).cuda()
        k = pool[:, 1]
        for j, x in enumerate((math.nan, -math.nan, math.inf, -math.inf)):
            k[int(table[0, 4]), 3, 1, 10 + j] = x
            k[int(table[0, 5]), 12 + j % 4] = x   # token 90 .. is behind the end
        k[int(table[0, 4]), 5, 1, 10] = math.inf
        room = torch.full((n_pages, 3, 2, 64), 4.0, dtype=dtype, device="cuda")
        both = room[:, :2]
        want = R.bounds(k, both, table, length, starts)
        _same(A.page_bounds(k, both, table, length, starts), want, dtype)
        assert bool((room[:, 2] == 4).all()) and int(torch.isnan(want).sum()) == 4


def test_bounds_wrong_numbers(A):
    _say("bounds, wrong numbers")
    gen = torch.Generator().manual_seed(2)
    table, _, _, n_pages = _batch([(1, 100), (1, 100)], 16, gen)
    k = torch.randn((n_pages, 16, 2, 64), generator=gen).to(BF).cuda()
    for lens, starts in (([10 ** 9, 5], [0, 30, 50]), ([-4, 70], [-3, 2, 5]), ([50, 50], [0, 0, 0]), ([3, 2 ** 31 - 1], [0, 9, 2 ** 31 - 1])):
        out = torch.full((n_pages, 2, 2, 64), 9.0, dtype=BF, device="cuda")
        rows = (2 ** 31 - 1024) // 2
        want = R.bounds(k, out, table, _i32(lens), _i32(starts), rows)
        _same(A.page_bounds(k, out, table, _i32(lens), _i32(starts)), want, lens)
    empty = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    A.page_bounds(k, out, empty, _i32([]), _i32([0]))


# ---- selection ----------------------------------------------------------------------

def _select_case(lens, kv, group, d, t, dtype, *, seed=0, missing=0.0, kind="random"):
    gen = torch.Generator().manual_seed(seed)
    table, length, starts, n_pages = _batch(lens, t, gen, missing)
    rows = sum(q for q, _ in lens)
    q = torch.randn((rows, kv * group + 1, d), generator=gen).to(dtype).cuda()[:, :kv * group]
    middle, width = torch.randn((n_pages, 1, kv, d), generator=gen), torch.randn((n_pages, 1, kv, d), generator=gen).abs()
    b = torch.cat([middle - width, middle + width], 1)
    if kind == "few values":     # many equal scores
        q, b = (q * 2).round().clamp(-1, 1), (b[:, :, :, :1].round().clamp(-1, 1) + 0 * b)
    elif kind == "same pages":
        b = b[:1] + 0 * b
    elif kind == "near":         # scores that fp32 sums cannot tell apart: one step of one small column
        b = b[:1] + 0 * b
        b[:, :, :, 0] = torch.arange(n_pages)[:, None, None] % 200 * 2.0 ** -20
    elif kind == "zeros":
        b = 0 * b
    return dict(q=q, b=b.to(dtype).cuda().contiguous(), table=table, lens=length, starts=starts, t=t, kv=kv)


def _check_select(A, c, budget, sink, recent, what, **kw):
    out = torch.full((c["q"].shape[0], c["kv"], budget), -7, dtype=torch.int32, device="cuda")
    want = R.select(c["q"], c["b"], c["table"], c["lens"], c["starts"], c["t"], budget, sink, recent, out)
    got = A.select_pages(c["q"], c["b"], c["table"], c["lens"], c["starts"], page_tokens=c["t"], budget=budget, sink=sink,
                         recent=recent, out=out, **kw)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got.cpu(), want), (what, int((got.cpu() != want).sum()))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,group,d,t", [
    ([(1, 1)], 1, 1, 64, 16), ([(1, 3000), (1, 40), (0, 17), (1, 900)], 2, 4, 128, 16), ([(5, 700), (20, 300)], 3, 3, 96, 13),
    ([(70, 1000)], 1, 2, 80, 7), ([(2, 5000)], 1, 24, 128, 16), ([(1, 600)], 2, 70, 16, 1), ([(3, 900)], 1, 1, 256, 4),
    ([(130, 140), (1, 70)], 2, 1, 64, 1), ([(1, 20000)], 1, 8, 192, 8), ([(2, 500)] * 70, 1, 4, 128, 16)])
def test_select(A, lens, kv, group, d, t, dtype):
    _say("select", lens[:3], kv, group, d, t, dtype)
    for seed, (budget, sink, recent, missing, kind) in enumerate([
            (8, 1, 1, 0.0, "random"), (37, 3, 4, 0.2, "random"), (5, 0, 5, 0.0, "random"), (16, 1, 2, 0.1, "few values"),
            (12, 0, 1, 0.0, "near")]):
        c = _select_case(lens, kv, group, d, t, dtype, seed=seed, missing=missing, kind=kind)
        _check_select(A, c, budget, sink, recent, (lens[:3], seed), max_q_len=None if seed % 2 else 1)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,group,d,t", [
    ([(600, 900), (20, 300), (0, 40)], 8, 4, 128, 16), ([(260, 300)], 64, 1, 16, 16), ([(530, 700)], 4, 8, 64, 13),
    ([(850, 1000)], 5, 3, 96, 32), ([(515, 520)], 16, 2, 256, 16), ([(270, 300)], 8, 8, 128, 16), ([(260, 500)], 8, 4, 240, 16), ([(530, 1500)], 8, 4, 64, 1)])
def test_select_chunks(A, lens, kv, group, d, t, dtype):
    """Rows enough for blocks of tokens over pieces of the pages."""
    _say("select, chunks", lens, kv, group, d, t, dtype)
    kind = ("random", "near", "few values")[(kv + d // 16) % 3]
    c = _select_case(lens, kv, group, d, t, dtype, seed=d, missing=0.1, kind=kind)
    _check_select(A, c, 9, 1, 2, (lens, kind))


@pytest.mark.parametrize("kind", ["same pages", "zeros", "near", "few values"])
def test_select_where_many_scores_are_equal(A, kind):
    """More pages at the border than are ranked at once (256); tables in and beyond what the local memory holds."""
    _say("select, equal scores", kind)
    c = _select_case([(1, 1500), (2, 700)], 2, 2, 64, 1, BF, kind=kind)
    for budget, sink, recent in ((100, 0, 1), (600, 1, 1), (1400, 10, 50), (2, 1, 1)):
        _check_select(A, c, budget, sink, recent, (kind, budget))
    c = _select_case([(300, 320)], 32, 1, 16, 2, BF, kind=kind, missing=0.05)
    _check_select(A, c, 30, 1, 1, (kind, "chunk"))
    c = _select_case([(1, 13000)], 1, 1, 16, 1, FP, kind=kind, missing=0.05)
    _check_select(A, c, 400, 2, 3, (kind, "long"))


def test_select_large_and_odd_numbers(A):
    """Numbers whose sums pass fp32, infinities and NaN in bounds and queries, numbers below fp32's smallest."""
    _say("select, odd numbers")
    for dtype, big in ((BF, 3e38), (FP, 6e4)):
        for kind in range(6):
            c = _select_case([(1, 900), (3, 400)], 2, 3, 64, 2, dtype, seed=kind)
            b, q, gen = c["b"], c["q"], torch.Generator().manual_seed(kind)
            at = torch.randint(0, b.shape[0], (30,), generator=gen).cuda()
            if kind == 0:
                b.mul_(big / 8)
                q.mul_(big / 8)
            elif kind == 1:
                b[at[:10], 1, :, 5], b[at[10:20], 0, :, 6], b[at[20:], 0, 1] = math.inf, -math.inf, math.nan
            elif kind == 2:
                q[0, 1, 3], q[1, 4], q[2] = math.nan, math.inf, -0.0
            elif kind == 3:
                b.mul_(2.0 ** -100 if dtype == BF else 2.0 ** -16)
                q.mul_(2.0 ** -60 if dtype == BF else 2.0 ** -14)
            elif kind == 4:
                b[at] *= big / 8
            elif kind == 5:
                b[at[:10], 1, :, 5], q[:, :, 5] = math.inf, 0.0
            _check_select(A, c, 40, 1, 2, (dtype, kind))


def test_select_wrong_numbers_and_nothing(A):
    _say("select, wrong numbers")
    c = _select_case([(6, 300), (4, 200)], 2, 2, 64, 16, BF)
    for lens, starts in (([10 ** 9, -5], [0, 6, 10]), ([3, 90], [2, 7, 99]), ([100, 100], [0, 0, 0])):
        c["lens"], c["starts"] = _i32(lens), _i32(starts)
        _check_select(A, c, 9, 1, 1, lens)
    c["table"] = torch.full_like(c["table"], -1)
    c["lens"], c["starts"] = _i32([300, 200]), _i32([0, 6, 10])
    _check_select(A, c, 4, 1, 1, "no page")
    c["q"] = c["q"][:0]
    assert A.select_pages(c["q"], c["b"], c["table"], c["lens"], _i32([0, 0, 0]), page_tokens=16, budget=4).shape == (0, 2, 4)


def test_select_rows_that_see_no_page(A):
    """Beside long contexts, few rows and many: their lists are all -1."""
    _say("select, rows without pages")
    for lens in ([(1, 0), (1, 20000), (3, 2)], [(40, 0), (200, 20000), (30, 17)]):
        _check_select(A, _select_case(lens, 4, 2, 64, 16, BF), 9, 1, 2, lens)


# ---- attention over selected pages ---------------------------------------------------

def _attend_case(lens, kv, group, d, t, dtype, listed, *, seed=0, missing=0.0):
    gen = torch.Generator().manual_seed(seed)
    table, length, starts, n_pages = _batch(lens, t, gen, missing)
    rows = sum(q for q, _ in lens)
    q = torch.randn((rows, kv * group + 2, d), generator=gen).to(dtype).cuda()[:, :kv * group]
    k, v = (torch.randn((n_pages, t, kv, d), generator=gen).to(dtype).cuda() for _ in range(2))
    picked = torch.randint(-2, table.shape[1] + 2, (rows, kv, listed), generator=gen).int()
    if seed % 3:   # ascending, and now and then not
        picked = torch.where(torch.rand((rows, kv, 1), generator=gen) < 0.1, picked, picked.sort(-1).values)
    return dict(q=q, k=k, v=v, table=table, lens=length, starts=starts, picked=picked.cuda())


def _attend(A, c, **kw):
    return A.selected_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], c["picked"], return_lse=True, **kw)


def _reference(c, scale=None):
    return R.selected(*(c[x] for x in ("q", "k", "v", "table", "lens", "starts", "picked")), scale or c["q"].shape[2] ** -0.5)


def _check_selected(A, c, what, **kw):
    out, lse = _attend(A, c, **kw)
    want = _reference(c, kw.get("scale"))
    _close(out, want[0], want[2], (what, "out"))
    _close(lse, want[1], want[3], (what, "lse"))
    return out, lse


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,group,d,t,listed", [
    ([(1, 1)], 1, 1, 64, 16, 1), ([(1, 3000), (1, 40), (0, 17), (1, 900)], 2, 4, 128, 16, 40), ([(5, 700), (20, 300)], 3, 3, 96, 13, 7),
    ([(1, 600)], 2, 40, 16, 1, 100), ([(3, 900)], 1, 1, 256, 4, 33), ([(300, 1000), (1, 9)], 5, 2, 64, 64, 3), ([(250, 500)], 5, 1, 256, 16, 2),
    ([(1, 20000)], 1, 8, 192, 8, 500), ([(2, 500)] * 70, 8, 4, 112, 16, 3), ([(1, 5000)], 1, 17, 128, 100, 30),
    ([(300, 900), (250, 250)], 8, 4, 128, 16, 5), ([(520, 1300)], 8, 4, 64, 64, 4), ([(1100, 1111)], 8, 2, 128, 1, 30),
    ([(300, 700), (0, 9), (260, 1100)], 8, 4, 256, 13, 6), ([(700, 2000)], 12, 2, 96, 100, 3), ([(150, 3000)], 3, 37, 128, 32, 20)])
def test_selected(A, lens, kv, group, d, t, listed, dtype):
    _say("selected", lens[:3], kv, group, d, t, listed, dtype)
    for seed, missing in enumerate((0.0, 0.15, 0.0)):
        if seed == 0 and sum(q for q, _ in lens) > 400:
            continue   # lists in any order of many rows: the ascending ones with some that are not are enough
        c = _attend_case(lens, kv, group, d, t, dtype, listed, seed=seed, missing=missing)
        _check_selected(A, c, (lens[:3], seed), **({"scale": 0.3} if seed else {}))


def test_selected_nothing_twice_and_far_outside(A):
    _say("selected, odd lists")
    c = _attend_case([(3, 200), (2, 90)], 2, 2, 64, 16, BF, 6, seed=5)
    c["picked"][0] = -1
    c["picked"][1, 0] = _i32([2, 2, 1 << 20, 0, 2, 5])
    c["picked"][2, 1] = _i32([2 ** 31 - 1, -2 ** 31, 1 << 27, 13, 12, 12])
    c["picked"][3] = 5   # pages behind the sequence's end
    out, lse = _check_selected(A, c, "odd lists")
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())


def test_all_pages_listed_is_paged_attention(A):
    _say("selected, all pages")
    for lens, dtype in (([(1, 700), (1, 33)], BF), ([(90, 400), (200, 300)], FP)):
        c = _attend_case(lens, 4, 2, 128, 16, dtype, 50, seed=6)
        c["picked"] = torch.arange(50, dtype=torch.int32, device="cuda").expand(c["picked"].shape).contiguous()
        out, lse = _check_selected(A, c, "all")
        full = A.paged_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], return_lse=True)
        want = _reference(c)
        _close(out, full[0].cpu().double(), 2 * want[2], "all, out")
        _close(lse, full[1].cpu().double(), 2 * want[3], "all, lse")


def test_selected_numbers_that_are_not_seen(A):
    """NaN and infinities behind a row's own token, in pages that are not listed, and in those that are."""
    _say("selected, NaN and infinities")
    c = _attend_case([(4, 100), (1, 60)], 2, 2, 64, 16, BF, 4, seed=7)
    c["picked"][:4] = _i32([0, 3, 6, -1])
    c["picked"][4:] = _i32([1, 2, 3, 3])
    for page, token in ((6, 3), (6, 4), (1, 0), (6, 8)):   # tokens 99, behind the end; 100; a page not listed; behind the end
        for pool, x in ((c["k"], math.nan), (c["v"], math.inf)):
            pool[int(c["table"][0, page]), token] = x
    c["v"][int(c["table"][0, 3]), 2, 1, 5] = -math.inf
    c["v"][int(c["table"][0, 3]), 4, 0, 6] = math.nan
    out, lse = _attend(A, c)
    want = _reference(c)
    bad = torch.isnan(want[1])
    assert bool(bad[3].all()) and not bool(bad[:3].any())   # the row that sees token 99
    for g, w, tol in ((out, want[0], want[2]), (lse, want[1], want[3])):
        g = g.cpu().double()
        keep = ~bad[..., None].expand_as(w) if w.dim() == 3 else ~bad
        assert bool(((g == w) | (torch.isnan(g) & torch.isnan(w)) | ((g - w).abs() <= tol))[keep].all())


def test_selected_numbers_that_others_see(A):
    """Blocks of rows with lists of their own: NaN and infinities of V reach the rows that list their pages and no other of
    the block, and where there are none the block is done once."""
    _say("selected, NaN and infinities in blocks")
    for d, t, dtype in ((128, 16, BF), (64, 13, FP)):
        c = _attend_case([(300, 700), (260, 500)], 8, 4, d, t, dtype, 6, seed=10)
        for page, token, pool, x in ((3, 2, "v", math.nan), (7, 1, "v", math.inf), (9, 0, "v", -math.inf), (5, 4, "k", math.nan),
                                     (7, 3, "v", math.inf)):
            c[pool][int(c["table"][0, page]), token, page % 8, 5] = x
        for s, total in ((0, 700), (1, 500)):   # behind the end
            if total % t:
                for pool in ("k", "v"):
                    c[pool][int(c["table"][s, total // t]), total % t:] = math.nan
        out, lse = _attend(A, c)
        want = _reference(c)
        bad = torch.isnan(want[1])
        assert bool(bad.any()) and bool(torch.isinf(want[0]).any()) and bool(torch.isnan(want[0])[~bad].any())
        for g, w, tol in ((out, want[0], want[2]), (lse, want[1], want[3])):
            g = g.cpu().double()
            keep = ~bad[..., None].expand_as(w) if w.dim() == 3 else ~bad
            assert bool(((g == w) | (torch.isnan(g) & torch.isnan(w)) | ((g - w).abs() <= tol))[keep].all()), d


def test_selected_wrong_numbers_stay_inside(A):
    _say("selected, wrong numbers")
    c = _attend_case([(6, 60), (10, 200)], 2, 4, 128, 16, BF, 5, seed=8)
    c["lens"], c["starts"] = _i32([3, 10 ** 6]), _i32([2, 7, 99])
    out = torch.full_like(c["q"], 7.0).contiguous()
    got, _ = _attend(A, c, out=out)
    want = _reference(c)
    assert bool((got[:2] == 7).all())
    _close(got[2:], want[0][2:], want[2][2:], "wrong numbers")


# ---- together -----------------------------------------------------------------------

def test_a_serving_loop(A):
    """Steps as an engine runs them: pages for the new tokens, append, bounds, selection, attention over the selected pages,
    then a draft as a tree whose rejected part is given back; results against the formulas, and the same captured."""
    _say("serving loop")
    gen = torch.Generator(device="cuda").manual_seed(3)
    kv, g, d, t, seqs, n_pages, cols = 2, 4, 128, 16, 3, 90, 40
    heads = kv * g
    k_pages, v_pages = (torch.zeros((n_pages, t, kv, d), dtype=BF, device="cuda") for _ in range(2))
    bounds = torch.zeros((n_pages, 2, kv, d), dtype=BF, device="cuda")
    table, lens = torch.full((seqs, cols), -1, dtype=torch.int32, device="cuda"), _i32([0] * seqs)
    free, n_free = torch.arange(n_pages, dtype=torch.int32, device="cuda").flip(0).contiguous(), _i32([n_pages])
    rope = A.rope_table(4096, 64)

    def step(wanted, rows, x):
        plan = A.allot_pages(table, lens, wanted, free, n_free, page_tokens=t, max_rows=rows, in_place=True)
        q = A.append_tokens(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], k_pages, v_pages, plan.slots, plan.positions, rope)
        A.page_bounds(k_pages, bounds, table, lens, plan.q_starts)
        return plan, q

    def sparse(wanted, rows, x):
        plan, q = step(wanted, rows, x)
        picked = A.select_pages(q, bounds, table, lens, plan.q_starts, page_tokens=t, budget=6, sink=1, recent=2)
        return plan, q, picked, A.selected_attention(q, k_pages, v_pages, table, lens, plan.q_starts, picked, return_lse=True)

    def check(plan, q, picked, result):
        n = int(plan.q_starts[-1])
        want = R.select(q, bounds, table, lens, plan.q_starts, t, 6, 1, 2, picked)
        assert torch.equal(picked.cpu()[:n], want[:n])
        want = R.selected(q, k_pages, v_pages, table, lens, plan.q_starts, picked, d ** -0.5)
        _close(result[0][:n], want[0][:n], want[2][:n], "loop, out")
        _close(result[1][:n], want[1][:n], want[3][:n], "loop, lse")

    rand = lambda n: torch.randn((n, heads + 2 * kv, d), generator=gen, device="cuda").to(BF)  # noqa: E731
    check(*sparse(_i32([200, 77, 390]), 700, rand(700)))            # prompts; the rows behind the last are padding
    for _ in range(3):
        check(*sparse(_i32([1, 1, 1]), 3, rand(3)))
    # a draft of 7 tokens: the root, two children, four grandchildren
    parents = [-1, 0, 0, 1, 1, 2, 2]
    line = []
    for i, p in enumerate(parents):
        line.append((line[p] if p >= 0 else 0) | 1 << i)
    mask = torch.tensor(line * seqs, device="cuda")[:, None]
    held = lens.clone()
    plan, q = step(_i32([7, 7, 7]), 21, rand(21))
    out, lse = A.tree_attention(q, k_pages, v_pages, table, lens, plan.q_starts, mask, return_lse=True)
    want = R.tree(q, k_pages, v_pages, table, lens, plan.q_starts, mask, d ** -0.5)
    _close(out, want[0], want[2], "loop, tree")
    _close(lse, want[1], want[3], "loop, tree lse")
    # the line 0, 2, 5 is accepted: its keys and values move to the front, the other tokens' pages go back
    for pool in (k_pages, v_pages):
        flat = pool.flatten(0, 1)
        slots = plan.slots.reshape(seqs, 7)
        flat[slots[:, [1, 2]].reshape(-1)] = flat[slots[:, [2, 5]].reshape(-1)]
    lens.copy_(held + 3)
    back = A.release_pages(table, lens, free, n_free, page_tokens=t, in_place=True)
    used = int(((lens + t - 1) // t).sum())
    assert int(n_free) == n_pages - used and int(back.n_released.sum()) == sum(
        -(-(int(x) + 7) // t) + -(-(int(x) + 3) // t) * -1 for x in held)
    # captured decoding steps against eager ones on the same state
    wanted, x = _i32([1, 1, 1]), rand(3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    state = (table, lens, free, n_free, k_pages, v_pages, bounds)
    start = [y.clone() for y in state]
    with torch.cuda.stream(stream):
        sparse(wanted, 3, x)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sparse(wanted, 3, x)
    for y, z in zip(state, start):
        y.copy_(z)
    for _ in range(4):
        x.copy_(rand(3))
        before = [y.clone() for y in state]
        want = sparse(wanted, 3, x)
        want = (want[2].clone(), want[3][0].clone(), want[3][1].clone(), *(y.clone() for y in state))
        for y, z in zip(state, before):
            y.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((got[2], *got[3], *state), want):
            assert torch.equal(a, b)
        check(*got)


def test_tensors_that_are_written_have_a_new_version(A):
    _say("versions")
    c = _attend_case([(2, 40)], 2, 2, 64, 16, BF, 2)
    bounds, out, picked = torch.zeros((c["k"].shape[0], 2, 2, 64), dtype=BF, device="cuda"), torch.empty_like(c["q"]).contiguous(), c["picked"]
    table, free, n_free, lens = c["table"].clone(), _i32([1, 2, 3]), _i32([3]), c["lens"].clone()
    batch, mask = (c["table"], c["lens"], c["starts"]), torch.ones((2, 1), dtype=torch.int64, device="cuda")
    for written, call in (((bounds,), lambda: A.page_bounds(c["k"], bounds, *batch)),
                          ((picked,), lambda: A.select_pages(c["q"], bounds, *batch, page_tokens=16, budget=2, out=picked)),
                          ((out,), lambda: A.selected_attention(c["q"], c["k"], c["v"], *batch, picked, out=out)),
                          ((out,), lambda: A.tree_attention(c["q"], c["k"], c["v"], *batch, mask, out=out)),
                          ((table,), lambda: A.allot_pages(table, lens, _i32([1]), free, n_free, page_tokens=16, max_rows=2)),
                          ((free,), lambda: A.release_pages(table, _i32([0]), free, n_free, page_tokens=16)),
                          ((table, lens, n_free), lambda: A.allot_pages(table, lens, _i32([1]), free, n_free, page_tokens=16, max_rows=2, in_place=True)),
                          ((table, free, n_free), lambda: A.release_pages(table, _i32([0]), free, n_free, page_tokens=16, in_place=True))):
        before = [t._version for t in written]
        call()
        assert all(t._version > x for t, x in zip(written, before))


@pytest.mark.parametrize("lens", [[(1, 700), (3, 400)], [(400, 900)]])
def test_pages_behind_four_gigabytes(A, lens):
    """Of a pool whose pages lie far apart: byte and element offsets pass 32 bits.  The same pages side by side give the
    same bits."""
    _say("far pages", lens)
    c = _attend_case(lens, 8, 4, 64, 16, BF, 5, seed=1)
    near, apart = c["k"].shape[0], 1 << 26                                # pages 128 MiB apart: 5 to 9 GiB
    n = min(near, 40)
    c["table"] = torch.where(c["table"] >= 0, c["table"] % n, c["table"])
    batch, d, t, kv = (c["table"], c["lens"], c["starts"]), 64, 16, 8

    def far(x, step):
        room = torch.empty((n - 1) * step + x[0].numel(), dtype=BF, device="cuda")
        y = room.as_strided((n, *x.shape[1:]), (step, *x[0].stride()))
        y.copy_(x[:n])
        return y

    def run(k, v, bounds):
        A.page_bounds(k, bounds, *batch)
        picked = A.select_pages(c["q"], bounds, *batch, page_tokens=t, budget=5)
        rows = c["q"].shape[0]
        mask = torch.full((rows, -(-rows // 64)), -1, dtype=torch.int64, device="cuda")
        return (bounds.contiguous(), picked, *A.selected_attention(c["q"], k, v, *batch, picked, return_lse=True),
                *A.tree_attention(c["q"], k, v, *batch, mask, return_lse=True))

    k, v = c["k"][:n].contiguous(), c["v"][:n].contiguous()
    b = torch.randn((n, 2, kv, d), generator=torch.Generator().manual_seed(4)).to(BF).cuda()
    want = run(k, v, b.clone())
    got = run(far(k, apart), far(v, apart), far(b, apart))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    torch.cuda.empty_cache()


def test_chunks_in_a_graph_and_on_two_streams(A):
    """Chunks' kernels replayed from a graph, and two calls under way at once, against calls one by one."""
    _say("chunks, graph and streams")
    cases = [_attend_case([(600, 900), (20, 300)], 8, 4, 128, 16, BF, 9, seed=s) for s in (1, 2)]
    for c in cases:
        c["b"] = torch.randn((c["k"].shape[0], 2, 8, 128), device="cuda").to(BF)

    def run(c):
        batch = (c["table"], c["lens"], c["starts"])
        picked = A.select_pages(c["q"], c["b"], *batch, page_tokens=16, budget=9, sink=1, recent=2)
        return picked, *A.selected_attention(c["q"], c["k"], c["v"], *batch, picked, return_lse=True)

    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, stream in zip(cases, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append([run(c) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
    graph, c = torch.cuda.CUDAGraph(), cases[0]
    with torch.cuda.graph(graph):
        result = run(c)
    for i in range(4):
        c["q"].copy_(torch.randn(c["q"].shape, device="cuda"))
        want = run(c)
        for x in result:
            x.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, want)), i
