"""GPU tests of the operators on hot pages at the edges of their ranges: the largest sizes, numbers that are not finite
in every place of a tile, and what torch keeps of tensors that are written in place."""
from __future__ import annotations

import pytest
import torch

import hot_reference as R
from test_gpu_hot_ops import A, BF, FP, _attend, _batch, _check_attend, _check_mass, _close, _say  # noqa: F401  (A: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
def test_accounts_of_a_length_a_page_short_of_2_31(A, new):
    """Pages of 3,000 tokens and a table of as many as a call takes: the length and a page's tokens together pass 2^31.
    All pages but the last of the first sequence are cold; nothing in front of the accounts is written."""
    _say("accounts near 2^31", new)
    t, d = 3000, 16
    mp = (2 ** 31 - 1024) // t
    gen = torch.Generator(device="cuda").manual_seed(new)
    kp = torch.randn((2, t, 1, d), generator=gen, device="cuda").to(BF)
    q = torch.randn((2 * new, 1, d), generator=gen, device="cuda").to(BF)
    table = torch.full((2, mp), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    table[1, 0] = 0
    lens = torch.tensor([2 ** 31 - 1, 2000], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    mass = torch.rand((2, 1, mp), generator=gen, device="cuda")
    guard = torch.full((2 * mass.numel(),), 7.0, device="cuda")
    out = guard[mass.numel():].view(mass.shape)
    # the first sequence's rows see its last page as they would see the only page of a sequence of 3,000 tokens
    small, short = torch.tensor([[1], [0]], dtype=torch.int32), torch.tensor([t, 2000], dtype=torch.int32)
    _, lse, _, _ = R.attention(q, kp, kp, small, short, starts, d ** -0.5)
    lse = lse.float().cuda()
    A.attention_mass(q, lse, kp, table, lens, starts, mass, decay=0.5, max_q_len=new, out=out)
    ends = torch.stack([mass[0, :, -1:], mass[1, :, :1]])
    want, tol = R.attention(q, kp, None, small, short, starts, d ** -0.5, (lse, ends, 0.5))
    _close(torch.stack([out[0, :, -1:], out[1, :, :1]]), want, tol, new)
    assert torch.equal(out[0, :, :-1], 0.5 * mass[0, :, :-1]) and torch.equal(out[1, :, 1:], 0.5 * mass[1, :, 1:])
    assert bool((guard[:mass.numel()] == 7).all())


def _spoil(b, bad, t, tile):
    """``bad`` in V's last head at tokens around the first new one of every sequence of several, each in a column of its
    own: new tokens, the ones before them in the same tile of ``tile`` keys, others, and one beside a cold page."""
    new = (b["starts"][1:] - b["starts"][:-1]).tolist()
    for s, length in enumerate(b["lens"].tolist()):
        if new[s] == 0:
            continue
        sees = length - new[s] + 1                             # tokens that the first row sees
        tiles = [sees // w * w for w in (tile, 32, 64)]
        at = [sees - 1, sees, length - 1, length - 2, sees - 2, sees - 7, 0, 5, *tiles, *(x - 1 for x in tiles),
              *(x + 3 for x in tiles), length // 2]
        if length > 200:
            b["table"][s, 16 // t] = -1                        # the pages of tokens 16 to 31 are cold
        for c, token in enumerate(dict.fromkeys(at)):
            page = int(b["table"][s, token // t]) if 0 <= token < length else -1
            if page >= 0:
                b["vp"][page, token % t, -1, c] = bad


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("lens", [[(3, 40)], [(2, 33), (1, 70), (4, 300)], [(150, 150)], [(150, 333), (1, 64)], [(5, 5001)],
                                  [(150, 3500)]])
def test_numbers_that_rows_see_reach_them(A, lens, d, bad):
    """An infinity or a NaN in V reaches every row that sees its token, wherever in a tile the token is, and no other row,
    column or head: sequences of few and of many rows, whole and in pieces, with cold pages."""
    _say("seen", lens, d, bad)
    for dtype, t, group in ((BF, 16, 2), (FP, 8, 3)):
        b = _batch(lens, group, 2, d, t, dtype, seed=d)
        _spoil(b, bad, t, 64 if d <= 128 else 32)
        for hint in (True, False):
            _check_attend(A, b, (lens, d, bad, dtype, hint), hint)


# A launch has fewer than 2^32 threads, 2^24 workgroups of 256: calls of more.

def test_an_append_of_more_tokens_than_a_launch_has_threads_for(A):
    _say("append of 2^26 tokens")
    n, d = 2 ** 26 + 5, 16
    k = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1, 1).repeat(1, 1, 8).view(BF).view(n, 1, d)
    pages = torch.zeros((n, 1, 1, d), dtype=BF, device="cuda")
    empty = torch.zeros((n, 0, d), dtype=BF, device="cuda")
    slots = torch.arange(n - 1, -1, -1, device="cuda")
    A.append_tokens(empty, k, None, pages, None, slots, torch.zeros(n, dtype=torch.int32, device="cuda"), A.rope_table(1, 0))
    # numbers pass through fp32, which turns a NaN whose first mantissa bit is 0 into one where it is 1; all else is exact
    got, want = pages[:, 0], k.flip(0)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert bool(((got.view(torch.int16) == want.view(torch.int16)) | nan).all())


@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_more_sequences_and_heads_than_a_launch_has(A, new):
    """The joins of the pieces: workgroups for every sequence and head (few rows), and for eight rows of these (many).
    All sequences but three have no new tokens, among them the last one, which is in pieces."""
    _say("joins of 2^24 workgroups", new)
    heads, t, d, seqs = 256, 16, 16, 65537 if new == 1 else 4097
    gen = torch.Generator(device="cuda").manual_seed(new)
    mp, some = 64, [3, seqs // 2, seqs - 1]
    kp = torch.randn((3 * mp, t, heads, d), generator=gen, device="cuda").to(BF)
    vp = torch.randn((3 * mp, t, heads, d), generator=gen, device="cuda").to(BF)
    table = torch.full((seqs, mp), -1, dtype=torch.int32, device="cuda")
    table[some] = torch.randperm(3 * mp, generator=gen, device="cuda").int().view(3, mp)
    lens, count = torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda")
    lens[some] = torch.tensor([60, 700, mp * t - 5], dtype=torch.int32, device="cuda")
    count[some] = torch.tensor([1, 1, new], dtype=torch.int32, device="cuda")
    starts = torch.cat([count.new_zeros(1), count.cumsum(0).int()])
    q = torch.randn((2 + new, heads, d), generator=gen, device="cuda").to(BF)
    out, lse = A.paged_attention(q, kp, vp, table, lens, starts, max_q_len=new, return_lse=True)
    few = torch.cat([starts[[s]] for s in some] + [starts[-1:]])
    want, wl, tol, ltol = R.attention(q, kp, vp, table[some], lens[some], few, d ** -0.5)
    _close(out, want, tol, "out")
    _close(lse, wl, ltol, "lse")


def test_accounts_of_more_tiles_than_a_launch_has(A):
    """A chunk at the end of a wide table beside thousands of sequences without new tokens, all accounts in place."""
    _say("accounts of 2^24 workgroups")
    heads, t, d, seqs, mp, new = 2, 64, 64, 4097, 2049, 40
    gen = torch.Generator(device="cuda").manual_seed(3)
    kp = torch.randn((4, t, heads, d), generator=gen, device="cuda").to(BF)
    table = torch.full((seqs, mp), -1, dtype=torch.int32, device="cuda")
    table[-1, [0, 1000, mp - 2, mp - 1]] = torch.tensor([2, 0, 3, 1], dtype=torch.int32, device="cuda")
    lens = torch.full((seqs,), 500, dtype=torch.int32, device="cuda")
    lens[-1] = mp * t - 3
    starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    starts[-1] = new
    q = torch.randn((new, heads, d), generator=gen, device="cuda").to(BF)
    _, lse, _, _ = R.attention(q, kp, kp, table[-1:], lens[-1:], starts[-2:], d ** -0.5)
    lse = lse.float().cuda()
    mass = torch.rand((seqs, heads, mp), generator=gen, device="cuda")
    before = mass.clone()
    A.attention_mass(q, lse, kp, table, lens, starts, mass, out=mass)
    want, tol = R.attention(q, kp, None, table[-1:], lens[-1:], starts[-2:], d ** -0.5, (lse, before[-1:], 1.0))
    _close(mass[-1:], want, tol, "accounts")
    assert torch.equal(mass[:-1], before[:-1])


def test_an_eviction_of_more_sequences_than_a_launch_has(A):
    _say("eviction of 2^24 sequences")
    seqs = 2 ** 24 + 3
    table = torch.arange(2 * seqs, dtype=torch.int32, device="cuda").view(seqs, 2)
    mass = torch.rand((seqs, 1, 2), device="cuda")
    lens = torch.full((seqs,), 20, dtype=torch.int32, device="cuda")
    e = A.evict_pages(mass, table, lens, page_tokens=16, budget=1, sink=0)
    assert bool((e.n_evicted == 1).all()) and bool((e.kv_lens == 4).all())
    assert torch.equal(e.evicted[:, 0], table[:, 0]) and torch.equal(e.page_table[:, 0], table[:, 1])
    assert torch.equal(e.mass[:, 0, 0], mass[:, 0, 1]) and bool((e.page_table[:, 1] == -1).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("which", ["q", "k"])
def test_a_row_without_a_weight_reaches_the_pages_it_sees_only(A, which, d):
    """A NaN in one new token's query, or in its key, makes its rows' log-sum-exp NaN (and those of the rows behind it,
    for the key): the pages that these rows see have NaN accounts of that head, all others the 64-bit form's."""
    _say("NaN rows", which, d)
    for lens in ([(4, 300)], [(150, 400), (1, 60)], [(200, 200)]):
        for token in (1, lens[0][0] // 2):
            b = _batch(lens, 3, 2, d, 16, BF, seed=d)
            key = lens[0][1] - lens[0][0] + token
            if which == "q":
                b["q"][token, 4] = float("nan")                # a head of the second KV head
            else:
                b["kp"][int(b["table"][0, key // 16]), key % 16, 1] = float("nan")
            for hint in (True, False):
                _, lse = _attend(A, b, hint)
                assert bool(torch.isnan(lse[token, 4])) and not bool(torch.isnan(lse[:, :3]).any())
                _check_mass(A, b, lse, (which, d, lens, token, hint), hint=hint)


def _serving_calls(A):
    """The tensors that each call writes, and the call."""
    b = _batch([(1, 40), (3, 70)], 4, 2, 128, 16, BF, seed=1)
    out, mass = torch.zeros_like(b["q"]), torch.zeros((2, 2, b["table"].shape[1]), device="cuda")
    _, lse = _attend(A, b)
    k, v = torch.randn((2, 4, 2, 128), device="cuda").to(BF)
    slots, pos, rope = torch.arange(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), A.rope_table(9, 64)
    rest = [b[x] for x in ("q", "kp", "vp", "table", "lens", "starts")]
    yield [b["q"], b["kp"], b["vp"]], lambda: A.append_tokens(b["q"], k, v, b["kp"], b["vp"], slots, pos, rope, q_out=b["q"])
    yield [out], lambda: A.paged_attention(*rest, out=out)
    yield [mass], lambda: A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass, out=mass)
    yield [mass, b["table"], b["lens"]], lambda: A.evict_pages(mass, b["table"], b["lens"], page_tokens=16, budget=2,
                                                               in_place=True)


def test_tensors_that_are_written_have_a_new_version(A):
    """torch tells by a tensor's version that one saved for a gradient has been overwritten since."""
    _say("versions")
    for written, call in _serving_calls(A):
        before = [t._version for t in written]
        call()
        assert all(t._version > x for t, x in zip(written, before))
    scale = torch.ones((), device="cuda", dtype=BF, requires_grad=True)
    written, call = next(_serving_calls(A))
    y = (scale * written[1]).sum()                             # saves the pages
    with torch.no_grad():
        call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_tensors_of_inference_mode_are_written(A):
    """They have no versions, inside and outside of that mode."""
    _say("inference mode")
    with torch.inference_mode():
        calls = list(_serving_calls(A))
        for _, call in calls:
            call()
    for written, call in calls:
        assert all(t.is_inference() for t in written)
        call()


@pytest.mark.parametrize("t", [16, 300])
@pytest.mark.parametrize("group", [5, 20])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_accounts_with_a_hint_too_small(A, d, group, t):
    """Sequences of many more rows than ``max_q_len`` says: the rows come again for every block of keys."""
    _say("accounts, hint", d, group, t)
    b = _batch([(70, 200), (33, 33), (1, 90), (41, 1000)], group, 2, d, t, BF, seed=8)
    _, lse = _attend(A, b)
    b["most"] = 1
    _check_mass(A, b, lse, (d, group, t))


def test_accounts_of_wrong_lengths_and_hints(A):
    """Lengths below 0 and behind the table, with rows that see nothing, and a hint that is too small."""
    _say("accounts, wrong lengths")
    b = _batch([(3, 50), (4, 60), (9, 70)], 4, 2, 64, 16, BF, seed=6)
    for lens in ([-5, 60, 2 ** 31 - 1], [0, 0, 0], [2, 3, 70]):
        b["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for most in (1, 100):
            b["most"] = most
            _, lse = _check_attend(A, b, (lens, most))
            _check_mass(A, b, lse, (lens, most))


def test_captured_chunks_and_evictions_of_long_tables(A):
    """A graph of chunks in pieces beside decoding sequences, their accounts and evictions from tables of 8,000 and 20,000
    pages, replayed as lengths and numbers change, beside eager calls."""
    _say("captured chunks")
    b = _batch([(1, 700), (60, 2100), (1, 90), (140, 1500)], 2, 1, 128, 16, FP, seed=8)
    mass = torch.zeros((4, 1, b["table"].shape[1]), device="cuda")
    long = [(torch.rand((2, 1, n), device="cuda"), torch.arange(2 * n, dtype=torch.int32, device="cuda").view(2, n),
             torch.tensor([n * 16, n * 8], dtype=torch.int32, device="cuda")) for n in (8000, 20000)]

    def step():
        out, lse = _attend(A, b)
        m = A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass, decay=0.5)
        return [out, lse, m, *(x for t in long for x in A.evict_pages(*t, page_tokens=16, budget=3000))]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        b["q"].normal_()
        b["lens"].copy_(torch.tensor([700 - i, 2100 - 500 * i, 90, 140 + 300 * i], dtype=torch.int32))
        for m, _, _ in long:
            m.uniform_()
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w), i
