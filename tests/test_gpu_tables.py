"""GPU tests of page tables kept on the device (allot_pages, release_pages) against their rules (tests/tables_reference.py).
All results are whole numbers and have to be equal."""
from __future__ import annotations

import pytest
import torch

import tables_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A(hip):
    import vlx_tee_amd.attention as A

    return A


def _say(*what):
    print("case", *what, flush=True)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _state(seqs, cols, page, max_len, max_q, *, seed, extra_free=0, one_q=0.0):
    """Sequences of random lengths whose pages are in the table, and a stack of free ones."""
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max_len + 1, (seqs,), generator=gen).int()
    wanted = torch.randint(0, max_q + 1, (seqs,), generator=gen).int()
    wanted[torch.rand(seqs, generator=gen) < one_q] = 1
    held = (lens + page - 1) // page
    need = (lens + wanted + page - 1) // page - held
    n = int(held.sum() + need.sum()) + extra_free
    ids = torch.randperm(n + 1, generator=gen).int()
    table, at = torch.full((seqs, cols), -1, dtype=torch.int32), 0
    for s in range(seqs):
        table[s, :held[s]] = ids[at:at + int(held[s])]
        at += int(held[s])
    free = ids[at:].clone()
    return table.cuda(), lens.cuda(), wanted.cuda(), free.cuda(), int(need.sum())


def _check_allot(A, table, lens, wanted, free, n_free, page, rows, counts=None, in_place=False, what=""):
    want = R.allot(table, lens, wanted, free, n_free, page, rows, counts)
    stack = free.clone()
    got = A.allot_pages(table, lens, wanted, free, n_free, page_tokens=page, max_rows=rows, next_positions=counts,
                        in_place=in_place)
    assert torch.equal(free, stack), what
    for name, g, w in zip(("page_table", *A.Allotment._fields), (table, *got), want):
        if name == "next_positions" and counts is None:
            assert g is None
            continue
        assert g.dtype == w.dtype and torch.equal(g.cpu(), w), (what, name)
    if in_place:
        assert got.kv_lens is lens and got.n_free is n_free and got.next_positions is counts
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs,cols,page,max_len,max_q", [
    (1, 1, 16, 0, 1), (1, 9, 16, 100, 40), (5, 30, 1, 20, 9), (64, 40, 16, 500, 1), (63, 300, 13, 700, 90),
    (1024, 40, 16, 300, 3), (1024, 40, 16, 300, 50), (1025, 40, 16, 300, 2), (3000, 20, 64, 900, 5), (7, 3, 1000, 1700, 1200),
    (2, 5000, 4, 9000, 10000)])
def test_allot(A, seqs, cols, page, max_len, max_q, in_place):
    _say("allot", seqs, cols, page, max_len, max_q, in_place)
    for seed, free_part, room in ((1, 1.0, 1.0), (2, 0.5, 1.0), (3, 1.0, 0.6), (4, 0.0, 1.3)):
        table, lens, wanted, free, need = _state(seqs, cols, page, max_len, max_q, seed=seed + seqs)
        rows = int(int(wanted.sum()) * room)
        counts = lens + 1000 if seed % 2 else None
        _check_allot(A, table, lens, wanted, free, _i32([int(need * free_part)]), page, rows, counts, in_place,
                     (seqs, seed))


def test_allot_where_only_some_wait(A):
    """More sequences than one turn adds up: those of the first that need pages wait, the others' rows close up."""
    _say("allot, waiting in an early turn")
    seqs = 9000
    lens = torch.full((seqs,), 5, dtype=torch.int32, device="cuda")
    lens[::7] = 16                                   # these need a page for the next token
    table = torch.arange(seqs * 2, dtype=torch.int32, device="cuda").reshape(seqs, 2).contiguous()
    wanted = torch.ones_like(lens)
    for rows in (seqs, seqs - 10, 3000):
        for free in (0, 50, 700, seqs):
            _check_allot(A, table.clone(), lens, wanted, torch.arange(seqs, dtype=torch.int32, device="cuda") + 10 ** 6, _i32([free]), 16,
                         rows, what=(rows, free))


def test_allot_wrong_numbers(A):
    """Negative and too large lengths and requests, a stack with fewer entries than n_free says, negative ids."""
    _say("allot, wrong numbers")
    for rows in (50, 5000):
        table = torch.arange(6 * 8, dtype=torch.int32, device="cuda").reshape(6, 8)
        free = _i32([5, -3, 7, -1, 9, 1 << 30])
        _check_allot(A, table, _i32([-5, 1000, 17, 128, 127, -2 ** 31]), _i32([3, 2, -7, 1, 1, 2 ** 31 - 1]), free, _i32([100]), 16,
                     rows, what="wrong")
        _check_allot(A, table.clone(), _i32([0, 0, 0, 0, 0, 0]), _i32([40] * 6), free, _i32([-4]), 16, rows, what="no stack")
        cold = table.clone()
        cold[2, 1] = -1   # the last page is cold: new tokens of it have no slot, those of the next page do
        got = _check_allot(A, cold, _i32([0, 0, 20, 0, 0, 0]), _i32([0, 0, 20, 0, 0, 0]), _i32([11, 12, 13]), _i32([3]), 16, rows)
        assert bool((got.slots[:12] == -1).all()) and bool((got.slots[12:20] >= 0).all())


def test_allot_one_large_page_and_none(A):
    _say("allot, page of 2^31 - 1100 tokens, no sequences, no rows")
    page = 2 ** 31 - 1100
    _check_allot(A, _i32([[4]]), _i32([page - 3]), _i32([3]), _i32([8]), _i32([1]), page, 10, what="large page")
    _check_allot(A, _i32([[-1]]), _i32([0]), _i32([3]), _i32([8]), _i32([1]), page, 5000, what="large page, empty")
    empty = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    for rows in (0, 7, 5000):
        _check_allot(A, empty, _i32([]), _i32([]), _i32([1, 2]), _i32([2]), 16, rows, what="no sequences")
        _check_allot(A, _i32([[1, -1]]), _i32([3]), _i32([0]), _i32([]), _i32([0]), 16, rows, what="nothing asked")


def test_allot_table_with_a_stride(A):
    _say("allot, strided table")
    table, lens, wanted, free, need = _state(40, 30, 16, 200, 60, seed=5)
    wide = torch.full((40, 50), 77, dtype=torch.int32, device="cuda")
    wide[:, :30] = table
    _check_allot(A, wide[:, :30], lens, wanted, free, _i32([need]), 16, int(wanted.sum()))
    assert bool((wide[:, 30:] == 77).all())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs,cols,page,max_len,capacity", [
    (1, 1, 16, 16, 5), (1, 5000, 16, 30000, 6000), (64, 40, 16, 500, 10 ** 4), (300, 257, 7, 1700, 10 ** 5), (17, 4097, 1, 4000, 10 ** 5),
    (17, 8200, 3, 9000, 40000), (3, 12300, 16, 10 ** 5, 12000)])
def test_release(A, seqs, cols, page, max_len, capacity, in_place):
    _say("release", seqs, cols, page, max_len, capacity, in_place)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed + seqs)
        table = torch.randint(-1, 1 << 20, (seqs, cols), generator=gen).int()
        table[torch.rand(seqs, cols, generator=gen) < 0.3] = -1
        wide = torch.full((seqs, cols + 3), 99, dtype=torch.int32, device="cuda")
        wide[:, :cols] = table.cuda()
        given = wide[:, :cols] if seed else table.cuda()
        lens = torch.randint(-20, max_len, (seqs,), generator=gen).int().cuda()
        lens[torch.rand(seqs, generator=gen).cuda() < 0.2] = 0
        free = torch.randint(0, 100, (capacity,), generator=gen).int().cuda()
        n_free = _i32([(0, capacity // 2, capacity + 9)[seed]])
        want = R.release(given, lens, free, n_free, page)
        before = given.clone()
        got = A.release_pages(given, lens, free, n_free, page_tokens=page, in_place=in_place)
        for name, g, w in zip((*A.Release._fields, "stack"), (*got, free), want):
            assert torch.equal(g.cpu(), w), (seed, name)
        assert torch.equal(given, got.page_table if in_place else before)
        assert bool((wide[:, cols:] == 99).all())


@pytest.mark.parametrize("seqs,cols", [(5000, 7), (1400, 9000), (60000, 1)])
def test_release_from_thousands(A, seqs, cols):
    """Counts that one workgroup adds up."""
    _say("release, thousands", seqs, cols)
    gen = torch.Generator(device="cuda").manual_seed(seqs)
    table = torch.randint(-9, 1 << 20, (seqs, cols), generator=gen, device="cuda").int()
    lens = torch.randint(0, 16 * cols, (seqs,), generator=gen, device="cuda").int()
    at = torch.arange(cols, device="cuda")[None]
    goes = (table >= 0) & (at >= ((lens + 15) // 16)[:, None])
    ids, all_of = table[goes], goes.sum(1).int()
    for capacity in (3 + ids.numel(), 3 + ids.numel() // 3):
        free = torch.full((capacity,), 77, dtype=torch.int32, device="cuda")
        given = table.clone()
        got = A.release_pages(given, lens, free, _i32([3]), page_tokens=16, in_place=True)
        fits = goes & ((goes.flatten().cumsum(0).reshape(seqs, cols) + 3) <= capacity)
        assert torch.equal(got.n_free, _i32([min(capacity, 3 + ids.numel())]))
        assert torch.equal(free[3:], ids[:capacity - 3]) and bool((free[:3] == 77).all())
        assert torch.equal(given, torch.where(fits, -1, table)) and torch.equal(got.n_released, fits.sum(1).int())
    assert torch.equal(A.release_pages(table, lens, torch.empty(4 + ids.numel(), dtype=torch.int32, device="cuda"), _i32([0]),
                                       page_tokens=16).n_released, all_of)


def test_release_nothing(A):
    empty = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    for n, want in ((2, 2), (9, 3), (-5, 0)):
        got = A.release_pages(empty, _i32([]), _i32([1, 2, 3]), _i32([n]), page_tokens=16)
        assert got.n_free.tolist() == [want] and got.n_released.numel() == 0
    got = A.release_pages(_i32([[3, 4]]), _i32([0]), _i32([]), _i32([0]), page_tokens=16)
    assert got.page_table.tolist() == [[3, 4]] and got.n_released.tolist() == [0]


@pytest.mark.parametrize("seqs,max_q", [(40, 3), (1500, 30)])
def test_steps_in_a_graph(A, seqs, max_q):
    """Captured in-place steps (more tokens, then a few sequences end), replayed with eager work between: every replay
    against the rules."""
    _say("graph", seqs, max_q)
    table, lens, wanted, free, need = _state(seqs, 400, 16, 100, max_q, seed=9, extra_free=60 * seqs)
    n_free, rows = _i32([free.numel()]), int(wanted.sum())
    kept = torch.where(torch.arange(seqs, device="cuda") % 7 == 3, 0, 1).int()
    state = (table, lens, free, n_free)
    start = [x.clone() for x in state]

    def step():
        got = A.allot_pages(table, lens, wanted, free, n_free, page_tokens=16, max_rows=rows, in_place=True)
        lens.mul_(kept)
        back = A.release_pages(table, lens, free, n_free, page_tokens=16, in_place=True)
        return got.slots, got.q_starts, back.n_released

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for x, y in zip(state, start):
        x.copy_(y)
    for turn in range(4):
        want = R.allot(table, lens, wanted, free, n_free, 16, rows)
        after = want[1] * kept.cpu()
        back = R.release(want[0], after, free, want[2], 16)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0].cpu(), want[4]) and torch.equal(out[1].cpu(), want[3]), turn
        for got, w in zip((table, n_free, out[2], free, lens), (*back, after)):
            assert torch.equal(got.cpu(), w), turn
        torch.ones(1000, device="cuda").sum().item()
