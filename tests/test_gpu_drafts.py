"""GPU tests of drafts as the guide has them: a tree's tokens take the positions of their depths, the accepted line moves to the
front of the draft's slots.  What is left then has to be what plain decoding of the accepted tokens leaves."""
from __future__ import annotations

import pytest
import torch

import sparse_reference as R

pytestmark = pytest.mark.gpu
KV, GROUP, D, T, SEQS = 2, 4, 128, 16, 3
HEADS = KV * GROUP
PARENTS = [-1, 0, 0, 1, 1, 2, 2]   # the root, two children, four grandchildren
DEPTH = [0, 1, 1, 2, 2, 2, 2]
LINE = [0, 2, 5]                   # accepted


@pytest.fixture(scope="module")
def A(hip):
    import vlx_tee_amd.attention as A

    return A


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _rand(n, seed, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, HEADS + 2 * KV, D), generator=gen, device="cuda").to(dtype)


class Engine:
    """Pools, a page table and a stack of free pages, as the guide sets them up."""

    def __init__(self, A, dtype, counted):
        pages = 60
        self.A, self.dtype = A, dtype
        self.k, self.v = (torch.zeros((pages, T, KV, D), dtype=dtype, device="cuda") for _ in range(2))
        self.bounds = torch.zeros((pages, 2, KV, D), dtype=dtype, device="cuda")
        self.table, self.lens = torch.full((SEQS, 20), -1, dtype=torch.int32, device="cuda"), _i32([0] * SEQS)
        self.free, self.n_free = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).contiguous(), _i32([pages])
        self.next = _i32([100, 0, 7]) if counted else None   # sequences that gave up pages before
        self.rope = A.rope_table(2048, 64)

    def append(self, wanted, x, depth=None):
        """depth: of a sequence's new tokens in their tree, None for a line."""
        plan = self.A.allot_pages(self.table, self.lens, _i32(wanted), self.free, self.n_free, page_tokens=T, max_rows=len(x),
                                  next_positions=self.next, in_place=True)
        positions = plan.positions
        if depth is not None:   # from a line's positions to the tree's
            positions = positions + _i32([d - i for i, d in enumerate(depth)]).repeat(SEQS)
        q = self.A.append_tokens(x[:, :HEADS], x[:, HEADS:HEADS + KV], x[:, HEADS + KV:], self.k, self.v, plan.slots, positions,
                                 self.rope)
        self.A.page_bounds(self.k, self.bounds, self.table, self.lens, plan.q_starts)
        return plan, q

    def accept(self, plan, held, line):
        """The line's keys and values to the front of the draft's slots; the lengths and counts of what was accepted."""
        slots = plan.slots.reshape(SEQS, -1)
        for pool in (self.k, self.v):
            flat = pool.flatten(0, 1)
            flat[slots[:, :len(line)].reshape(-1)] = flat[slots[:, line].reshape(-1)]
        drafted = slots.shape[1]
        self.lens.copy_(held + len(line))
        if self.next is not None:
            self.next -= drafted - len(line)

    def tokens(self, pool):
        """Every sequence's rows of a pool, in their order."""
        flat = pool.flatten(0, 1)
        out = []
        for s in range(SEQS):
            at = torch.arange(int(self.lens[s]), device="cuda")
            out.append(flat[self.table[s, at // T].long() * T + at % T])
        return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counted", [False, True])
def test_an_accepted_line_is_what_plain_decoding_leaves(A, dtype, counted):
    prompt, draft = _rand(36 + 15 + 61, 1, dtype), _rand(len(PARENTS) * SEQS, 2, dtype)
    per = draft.reshape(SEQS, len(PARENTS), HEADS + 2 * KV, D)
    tree, plain = Engine(A, dtype, counted), Engine(A, dtype, counted)
    for e in (tree, plain):
        e.append([36, 15, 61], prompt)
    bits = []
    for i, p in enumerate(PARENTS):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    mask = torch.tensor(bits * SEQS, device="cuda")[:, None]
    held = tree.lens.clone()
    plan, q = tree.append([len(PARENTS)] * SEQS, draft, DEPTH)
    batch = (tree.table, tree.lens, plan.q_starts)
    out, lse = A.tree_attention(q, tree.k, tree.v, *batch, mask, return_lse=True)
    want = R.tree(q, tree.k, tree.v, *batch, mask, D ** -0.5)
    assert bool(((out.cpu().double() - want[0]).abs() <= want[2]).all()) and bool(((lse.cpu().double() - want[1]).abs() <= want[3]).all())
    tree.accept(plan, held, LINE)
    # the same tokens one after another
    for nth, node in enumerate(LINE):
        step, one_q = plain.append([1] * SEQS, per[:, node].contiguous())
        rows = torch.arange(SEQS, device="cuda") * len(PARENTS) + node
        assert torch.equal(one_q, q[rows])                          # rotated by the same angles
        one, one_lse = A.paged_attention(one_q, plain.k, plain.v, plain.table, plain.lens, step.q_starts, return_lse=True)
        # both are within their bounds of the same numbers
        assert bool(((one.cpu().double() - want[0][rows.cpu()]).abs() <= want[2][rows.cpu()]).all()), nth
        assert bool(((one_lse.cpu().double() - want[1][rows.cpu()]).abs() <= want[3][rows.cpu()]).all()), nth
    assert torch.equal(tree.lens, plain.lens)
    for a, b in zip(tree.tokens(tree.k) + tree.tokens(tree.v), plain.tokens(plain.k) + plain.tokens(plain.v)):
        assert torch.equal(a, b)
    if counted:
        assert torch.equal(tree.next, plain.next)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_of_pages_that_moved_keys_fill(A, dtype):
    """The line ends with its page, which no later token enters: only a renewal brings the moved keys into the page's bounds."""
    e = Engine(A, dtype, False)
    e.append([29, 13, 61], _rand(29 + 13 + 61, 3, dtype))
    held = e.lens.clone()
    plan, _ = e.append([len(PARENTS)] * SEQS, _rand(len(PARENTS) * SEQS, 4, dtype), DEPTH)
    e.accept(plan, held, LINE)
    assert bool((e.lens % T == 0).all())
    A.release_pages(e.table, e.lens, e.free, e.n_free, page_tokens=T, in_place=True)
    want = R.bounds(e.k, torch.zeros_like(e.bounds), e.table, e.lens, torch.cat([e.lens.new_zeros(1), e.lens.cumsum(0)]).int())
    ids = torch.cat([e.table[s, :int(e.lens[s]) // T] for s in range(SEQS)]).long()

    def covers():
        return bool((e.bounds[ids, 0] <= want.cuda()[ids, 0]).all() and (e.bounds[ids, 1] >= want.cuda()[ids, 1]).all())

    assert not covers()   # what the draft left does not hold of the moved keys
    starts = torch.arange(SEQS + 1, dtype=torch.int32, device="cuda") * len(LINE)
    A.page_bounds(e.k, e.bounds, e.table, e.lens, starts)
    assert torch.equal(e.bounds[ids].cpu(), want[ids.cpu()])
