"""GPU tests of page selection and attention over selected pages at the ends of what one form of a kernel takes."""
from __future__ import annotations

import math

import pytest
import torch

import sparse_reference as R
from test_gpu_sparse import BF, FP, A, _attend, _attend_case, _check_select, _i32, _reference, _say, _select_case  # noqa: F401

pytestmark = pytest.mark.gpu


def _nan_as(c, what):
    """A row's log-sum-exp, and with it all of its result, is NaN exactly where the formula's is; other numbers as they are."""
    out, lse = _attend(A_, c)
    want = _reference(c)
    bad = torch.isnan(want[1])
    assert torch.equal(torch.isnan(lse.cpu()), bad), what
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want[0])), what
    return bad


@pytest.fixture(autouse=True)
def _module(A):
    global A_
    A_ = A


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,kv,group,d,t,listed", [
    ([(4, 100), (1, 60)], 2, 2, 64, 16, 4), ([(3, 900), (1, 500)], 2, 40, 128, 16, 20), ([(2, 700)], 1, 3, 256, 13, 9),
    ([(1200, 1300)], 1, 1, 64, 16, 3), ([(300, 700), (260, 500)], 8, 4, 128, 16, 6), ([(300, 700), (260, 500)], 8, 4, 96, 13, 6)])
def test_a_key_of_nan_makes_its_rows_nan(lens, kv, group, d, t, listed, dtype):
    """Few rows, rows one by one and blocks: a maximum that passes NaN over must not lose it."""
    _say("selected, keys of NaN", lens, kv, group, d, t)
    bad = []
    for seed in (1, 2):
        c = _attend_case(lens, kv, group, d, t, dtype, listed, seed=seed)
        for s, (_, n) in enumerate(lens):
            pages = -(-n // t)
            for page in (0, pages // 2, pages - 1):
                if page * t < n:
                    c["k"][int(c["table"][s, page]), 0, page % kv, 3] = math.nan
        bad.append(_nan_as(c, (lens, seed)))
    assert bool(torch.stack(bad).any()) and not bool(torch.stack(bad).all())


@pytest.mark.parametrize("columns", [11788, 11789, 12287, 12288, 12289])
def test_select_of_tables_at_the_local_memory_s_end(columns):
    _say("select, columns", columns)
    for lens in ([(1, columns)], [(257, columns)]) if columns in (12288, 12289) else ([(1, columns)],):   # a row a workgroup of 1,024, of 256
        c = _select_case(lens, 2, 1, 16, 1, BF, missing=0.02, seed=columns)
        _check_select(A_, c, 50, 1, 2, (columns, lens))


def test_bounds_of_more_rows_than_a_call_with_queries_takes():
    """Of 64 heads: sequences behind 2^31 / 64 rows of others have their pages' bounds too."""
    _say("bounds, many rows")
    gen = torch.Generator().manual_seed(1)
    k = torch.randn((9, 16, 64, 16), generator=gen).to(BF).cuda()
    table = torch.arange(9, dtype=torch.int32, device="cuda").repeat(2, 1).contiguous()
    bounds = torch.full((9, 2, 64, 16), 9.0, dtype=BF, device="cuda")
    lens, starts = _i32([0, 100]), _i32([0, 40_000_000, 40_000_100])
    want = R.bounds(k, bounds, table, lens, starts, 2 ** 31 - 1)
    assert torch.equal(A_.page_bounds(k, bounds, table, lens, starts).cpu(), want)


@pytest.mark.parametrize("kw", [dict(budget=1 << 31), dict(budget=1 << 62), dict(budget=0), dict(budget=(1 << 31) - 1, sink=1 << 31),
                                dict(budget=(1 << 31) - 1, recent=1 << 31), dict(budget=(1 << 31) - 1, sink=-1),
                                dict(budget=(1 << 31) - 1, sink=2 ** 63 - 1, recent=2 ** 63 - 1)])
def test_budgets_are_looked_at_before_anything_is_allocated(kw):
    _say("select, budgets", kw)
    c = _select_case([(300, 400)], 8, 1, 64, 16, BF)
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="budget"):
        A_.select_pages(c["q"], c["b"], c["table"], c["lens"], c["starts"], page_tokens=16, **kw)
    assert torch.cuda.max_memory_allocated() == held


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 256, 257, 320, 321, 385, 449, 512, 513, 576, 577, 640, 641, 705, 769, 833, 897, 961, 1023, 1024, 1025])
def test_select_of_tables_around_the_registers(pages):
    """Keys in as many registers as the table's columns need."""
    _say("select, pages", pages)
    c = _select_case([(3, 16 * pages), (2, 5 * pages)], 2, 3, 32, 16, FP, seed=pages, missing=0.05, kind=("random", "near", "few values")[pages % 3])
    for budget in (2, 40, 700):
        _check_select(A_, c, budget, 1, 1, (pages, budget))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,group", [([(1, 3000), (2, 1100)], 2), ([(2, 900), (3, 300)], 3), ([(1, 13000)], 1), ([(130, 1030)], 2)])
@pytest.mark.parametrize("kind", ["random", "near", "few values"])
def test_select_where_some_scores_are_no_numbers(lens, group, dtype, kind):
    """Fewer of these than are wanted, as many, and more, among scores that are finite, apart and equal: infinities of either
    sign in either bound, NaN, infinities that meet a query's 0, and sums that pass fp32 while all numbers are finite."""
    _say("select, some no numbers", lens, group, dtype, kind)
    for seed, bad in enumerate((1, 5, 40, 300) if lens[0][0] < 100 else (5, 300)):
        kv = 2 if len(lens) > 1 or lens[0][0] == 1 else 4
        c = _select_case(lens, kv, group, 32, 1, dtype, seed=seed, missing=0.03, kind=kind)
        gen = torch.Generator().manual_seed(seed)
        at = torch.randperm(c["b"].shape[0], generator=gen)[:bad * len(lens)].cuda()
        for j, (side, column, x) in enumerate([(1, 3, math.inf), (0, 4, -math.inf), (0, 5, math.nan), (1, 6, -math.inf), (0, 7, math.inf)]):
            c["b"][at[j::6], side, j % kv, column] = x
        if dtype == BF:
            c["b"][at[5::6], :, :, :] = 3e38
            c["q"][0, :, :8] = 2.0
        c["q"][-1, 0, 3] = 0.0
        many = sum(n for n, _ in lens) > 100   # (the reference takes its time)
        for budget in (7, 42) if many else (2, 7, 42, 320):
            _check_select(A_, c, budget, 1, 1, (lens, kind, bad, budget))
