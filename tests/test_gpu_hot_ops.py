"""GPU tests of the operators on hot pages (vlx-tee_amd/attention.py) against
their formulas in 64 bits (tests/hot_reference.py, which derives the bounds)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import hot_reference as R

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def A(hip):
    import vlx_tee_amd.attention as A

    return A


def _say(*what):
    print("case", *what, flush=True)


def _close(got, want, tol, what):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    ok = torch.isnan(want) | (got == want) | ((got - want).abs() <= tol)
    assert bool(ok.all()), (what, float((got - want).abs().nan_to_num(0, 0, 0).max()), int((~ok).sum()))


# ---- append ------------------------------------------------------------------------

def _append_case(A, n, heads, kv, d, r, t, dtype, *, interleaved=False, norm="full", strided=True, seed=0, single=False,
                 pages=None, interleaved_pool=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    parts = heads + kv * (1 if single else 2)
    x = torch.randn((n, parts, d), generator=gen, device="cuda").to(dtype)
    q, k = x[:, :heads], x[:, heads:heads + kv]
    v = None if single else x[:, heads + kv:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), None if single else v.contiguous()
    pages = pages or n // t + 3
    if interleaved_pool:   # K and V pages in turn, one buffer
        both = torch.full((pages, 2, t, kv, d), 9.0, dtype=dtype, device="cuda")
        kp, vp = both[:, 0], both[:, 1]
    else:
        kp = torch.full((pages, t, kv, d), 9.0, dtype=dtype, device="cuda")
        vp = None if single else torch.full((pages, t, kv, d), 9.0, dtype=dtype, device="cuda")
    slots = torch.randperm(pages * t, generator=gen, device="cuda")[:n]
    pos = torch.randint(0, 5000, (n,), generator=gen, device="cuda").int()
    rope = A.rope_table(5000, r)
    wl = {"full": (d, d), "tail": (0, d - r), "none": (0, 0), "q": (d, 0)}[norm]
    w = [(1 + 0.2 * torch.randn(m, generator=gen, device="cuda")).to(dtype) if m else None for m in wl]
    return dict(q=q, k=k, v=v, kp=kp, vp=vp, slots=slots, pos=pos, rope=rope, qw=w[0], kw=w[1], inter=interleaved)


def _run_append(A, c, **more):
    return A.append_tokens(c["q"], c["k"], c["v"], c["kp"], c["vp"], c["slots"], c["pos"], c["rope"], q_weight=c["qw"],
                           k_weight=c["kw"], eps=1e-5, interleaved=c["inter"], **more)


def _check_append(c, q_out, before_k, before_v, what):
    u = R.HALF[c["q"].dtype]
    pos, rope = c["pos"].cpu(), c["rope"].cpu()
    cpu = lambda x: None if x is None else x.cpu()  # noqa: E731

    def bound(want, big):   # the final rounding; squares, root, two products and a rotation in fp32 (fp16 results below 2^-14 step by 2^-24)
        return u * want.abs().nan_to_num(0) + (want.shape[-1] + 16) * 2.0 ** -24 * big.nan_to_num(0) + 2.0 ** -25

    want, big = R.rotated(c["q_in"].cpu(), cpu(c["qw"]), rope, pos, 1e-5, c["inter"])
    _close(q_out, want, bound(want, big), (what, "q"))
    want, big = R.rotated(c["k"].cpu(), cpu(c["kw"]), rope, pos, 1e-5, c["inter"])
    slots = c["slots"].cpu()
    ok = (slots >= 0) & (slots < c["kp"].shape[0] * c["kp"].shape[1])
    flat = c["kp"].cpu().flatten(0, 1)
    _close(flat[slots[ok]], want[ok], bound(want, big)[ok], (what, "k"))
    rest = torch.ones(flat.shape[0], dtype=torch.bool)
    rest[slots[ok]] = False
    assert torch.equal(flat[rest], before_k.flatten(0, 1)[rest]), (what, "other rows of K")
    if c["v"] is not None:
        fv = c["vp"].cpu().flatten(0, 1)
        assert torch.equal(fv[slots[ok]], c["v"].cpu()[ok]) and torch.equal(fv[rest], before_v.flatten(0, 1)[rest])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", [
    # n, q heads, kv heads, d, rope, page tokens
    (1, 8, 2, 128, 64, 16), (33, 32, 8, 128, 128, 16), (7, 15, 5, 96, 32, 13), (5, 3, 3, 80, 16, 7),
    (3, 4, 1, 64, 64, 1), (9, 6, 2, 192, 32, 29), (4, 2, 2, 256, 256, 64), (65, 1, 1, 16, 16, 5), (6, 2, 1, 32, 0, 16),
    (3, 2, 1, 1024, 512, 4), (2, 3, 1, 528, 112, 16), (40, 5, 3, 112, 48, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(A, shape, dtype, interleaved):
    _say("append", shape, dtype, interleaved)
    for norm in ("full", "none", "tail") if shape[4] not in (0, shape[3]) else ("full", "q"):
        c = _append_case(A, *shape, dtype, interleaved=interleaved, norm=norm, seed=sum(shape))
        bk, bv = c["kp"].cpu(), c["vp"].cpu()
        c["q_in"] = c["q"].clone()
        _check_append(c, _run_append(A, c), bk, bv, (shape, norm))


def test_append_latent_pages(A):
    _say("append latent 576")
    c = _append_case(A, 70, 16, 1, 576, 64, 64, BF, interleaved=True, norm="tail", single=True)
    bk, c["q_in"] = c["kp"].cpu(), c["q"].clone()
    _check_append(c, _run_append(A, c), bk, None, "latent")


def test_append_in_place_padding_and_unknown_positions(A):
    """q_out = q inside the projection's buffer; slots outside the pool write nothing; a position without angles gives
    NaN in the rotated columns only."""
    _say("append in place, padded")
    c = _append_case(A, 50, 8, 2, 128, 64, 16, BF, interleaved_pool=True)
    n_slots = c["kp"].shape[0] * 16
    c["slots"][[3, 4, 5, 6]] = torch.tensor([-1, n_slots, 1 << 40, -(1 << 40)], device="cuda")
    c["pos"][[7, 8]] = torch.tensor([-1, 5000], dtype=torch.int32, device="cuda")
    c["q_in"] = c["q"].clone()
    bk, bv, k_before = c["kp"].cpu(), c["vp"].cpu(), c["k"].clone()
    out = _run_append(A, c, q_out=c["q"])
    assert out.data_ptr() == c["q"].data_ptr() and torch.equal(c["k"], k_before)
    _check_append(c, out, bk, bv, "in place")
    assert torch.isnan(out[7, :, :64]).all() and torch.isfinite(out[7, :, 64:]).all()


def test_append_nothing(A):
    c = _append_case(A, 4, 8, 2, 128, 64, 16, BF)
    for x in ("q", "k", "v", "slots", "pos"):
        c[x] = c[x][:0]
    assert _run_append(A, c).shape == (0, 8, 128) and bool((c["kp"] == 9).all())


def test_append_same_slot_twice_is_one_of_them(A):
    _say("append, one slot for all tokens")
    c = _append_case(A, 64, 2, 2, 64, 32, 16, FP, strided=False)
    c["slots"].fill_(17)
    _run_append(A, c)
    row = c["vp"].flatten(0, 1)[17]
    for h in range(2):
        assert bool((c["v"][:, h] == row[h]).all(1).any())


# ---- batches -----------------------------------------------------------------------

def _batch(lens, group, kv, d, t, dtype, *, seed=0, missing=0.0, spread=1.0, extra_cols=0, pad_pages=0, stale=None):
    """lens: [(new tokens, tokens)].  Pages behind a sequence's tokens and rows behind its end hold ``stale``."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // t) for _, n in lens]
    mp, pages = max(max(need), 1) + extra_cols, sum(need) + 2
    ids = rng.permutation(pages)
    table = np.full((len(lens), mp), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    if missing:
        table[rng.random(table.shape) < missing] = rng.choice([-1, -7, pages, 2 ** 31 - 1])
    rows = sum(a for a, _ in lens)
    q = (spread * torch.randn((rows, group * kv, d), generator=gen, device="cuda")).to(dtype)
    shape = (pages, t, kv, d + pad_pages) if not pad_pages else (pages, t * kv * d + pad_pages)
    make = lambda: torch.randn(shape, generator=gen, device="cuda").to(dtype)  # noqa: E731
    kp, vp = make(), make()
    if pad_pages:
        kp, vp = (x[:, :t * kv * d].unflatten(1, (t, kv, d)) for x in (kp, vp))
    if stale is not None:
        for i, (_, n) in enumerate(lens):
            if n % t and table[i, n // t] in range(pages):
                kp[int(table[i, n // t]), n % t:] = stale
                vp[int(table[i, n // t]), n % t:] = stale
    return dict(q=q, kp=kp, vp=vp, table=torch.from_numpy(table).cuda(),
                lens=torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda"),
                starts=torch.tensor(np.cumsum([0] + [a for a, _ in lens]), dtype=torch.int32, device="cuda"),
                most=max(a for a, _ in lens), scale=d ** -0.5)


def _attend(A, b, hint=True, **more):
    return A.paged_attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], scale=b["scale"],
                             max_q_len=b["most"] if hint else None, return_lse=True, **more)


def _check_attend(A, b, what, hint=True):
    out, lse = _attend(A, b, hint)
    want, wl, tol, ltol = R.attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], b["scale"])
    _close(out, want, tol, (what, "out"))
    _close(lse, wl, ltol, (what, "lse"))
    return out, lse


def _check_mass(A, b, lse, what, decay=1.0, hint=True):
    gen = torch.Generator(device="cuda").manual_seed(5)
    mass = torch.rand((b["lens"].numel(), b["kp"].shape[2], b["table"].shape[1]), generator=gen, device="cuda")
    got = A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass, scale=b["scale"],
                           decay=decay, max_q_len=b["most"] if hint else None)
    want, tol = R.attention(b["q"], b["kp"], None, b["table"], b["lens"], b["starts"], b["scale"], (lse, mass, decay))
    _close(got, want, tol, (what, "mass"))


SHAPES = [(4, 2, 128, 16), (1, 3, 64, 7), (3, 5, 96, 13), (8, 1, 80, 1), (2, 1, 256, 64), (6, 2, 192, 100), (20, 1, 128, 16),
          (40, 1, 64, 16), (70, 1, 128, 16), (1, 1, 16, 3), (16, 2, 128, 300)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(A, shape, dtype):
    _say("decode", shape, dtype)
    lens = [(1, n) for n in (1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300, 777)]
    b = _batch(lens, *shape, dtype, seed=sum(shape), spread=2.0)
    out, lse = _check_attend(A, b, (shape, "decode"))
    _check_mass(A, b, lse, (shape, "decode"), decay=0.5)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("hint", [True, False])
def test_chunks(A, shape, dtype, hint):
    """Chunks at the end of a context, whole prompts, decoding and speculating sequences, empty ones, in one batch."""
    _say("chunks", shape, dtype, hint)
    lens = [(1, 700), (130, 130), (0, 50), (33, 257), (1, 1), (5, 300), (0, 0), (64, 64), (2, 129), (97, 513)]
    b = _batch(lens, *shape, dtype, seed=1 + sum(shape), spread=2.0)
    out, lse = _check_attend(A, b, (shape, hint), hint)
    _check_mass(A, b, lse, (shape, hint), hint=hint)


@pytest.mark.parametrize("most", [1, 2, 5, 9])
def test_long_contexts_in_pieces(A, most):
    _say("pieces", most)
    b = _batch([(most, 5001), (1, 40), (most, 9000)], 4, 2, 128, 16, BF, seed=most, spread=3.0)
    _, lse = _check_attend(A, b, most)
    _check_mass(A, b, lse, most)
    b = _batch([(most, 4111)], 12, 1, 64, 13, FP, seed=most, spread=3.0)
    _, lse = _check_attend(A, b, most)
    _check_mass(A, b, lse, most)


def test_prompt_over_a_long_context_in_pieces(A):
    _say("many rows in pieces")
    b = _batch([(150, 3500)], 2, 1, 128, 32, BF, seed=3, spread=2.0)
    _, lse = _check_attend(A, b, "pieces")
    _check_mass(A, b, lse, "pieces")


@pytest.mark.parametrize("lens", [[(1, 100), (1, 700)], [(40, 100), (200, 700), (1, 333)]])
@pytest.mark.parametrize("stale", [math.nan, math.inf, -math.inf, 3e4])
def test_missing_pages_and_stale_rows(A, lens, stale):
    """Pages that are not there take no part; neither does what stands behind a sequence's end."""
    _say("missing, stale", lens, stale)
    for dtype, missing in ((BF, 0.3), (FP, 0.0), (BF, 1.0)):
        b = _batch(lens, 4, 2, 128, 16, dtype, seed=7, missing=missing, stale=stale, extra_cols=3)
        out, lse = _check_attend(A, b, (lens, missing))
        _check_mass(A, b, lse, (lens, missing))
        if missing == 1.0:
            assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens", [[(3, 40)], [(150, 150)], [(150, 300), (1, 64)]])
def test_numbers_after_a_rows_token_do_not_reach_it(A, lens, bad):
    """A NaN or an infinity in the K or V of one new token reaches the rows that see it and no others."""
    _say("bad token", lens, bad)
    for which in ("kp", "vp"):
        b = _batch(lens, 2, 2, 128, 16, BF, seed=11)
        token = lens[0][1] - 2
        page = int(b["table"][0, token // 16])
        if which == "vp":
            b["vp"][page, token % 16, 1, 5] = bad
        else:
            b["kp"][page, token % 16, 1] = math.nan
        out, lse = _attend(A, b)
        want, wl, tol, ltol = R.attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], b["scale"])
        clean = torch.ones(out.shape[0], dtype=torch.bool)
        clean[lens[0][0] - 2:lens[0][0]] = False
        _close(out[clean.cuda()], want[clean], tol[clean], (lens, which, "clean rows"))
        _close(out[:, :2], want[:, :2], tol[:, :2], (lens, which, "other heads"))
        if which == "vp":
            other = [c for c in range(128) if c != 5]
            _close(out[..., other], want[..., other], tol[..., other], (lens, which, "other columns"))
            seen = out[lens[0][0] - 2:lens[0][0], 2:, 5].float().cpu()
            assert bool(torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all())
        else:
            assert bool(torch.isnan(out[lens[0][0] - 2:lens[0][0], 2:].float()).all())


def test_large_scores_and_equal_ones(A):
    """Scores far apart (one key takes all), and all equal."""
    _say("large scores")
    b = _batch([(1, 500), (64, 200)], 4, 2, 128, 16, BF, seed=2, spread=60.0)
    _check_attend(A, b, "large")
    b["q"].zero_()
    _, lse = _check_attend(A, b, "equal")
    _check_mass(A, b, lse, "equal")


def test_strides_pools_and_rows_of_no_sequence(A):
    """q inside a projection's output, padded pages, a slice of a wider table, rows before, between and behind the
    sequences left as they were."""
    _say("strides")
    b = _batch([(1, 90), (17, 60), (1, 333)], 4, 2, 128, 16, BF, seed=4, pad_pages=64, extra_cols=2)
    wide = torch.randn((b["q"].shape[0] + 5, 12, 128), device="cuda").to(BF)
    wide[2:-3, :8] = b["q"]
    b["q"] = wide[:, :8]
    b["starts"] += 2
    b["table"] = torch.cat([b["table"], b["table"]], 1)[:, :b["table"].shape[1]]
    out = torch.full(b["q"].shape, 7.0, dtype=BF, device="cuda")
    got, lse = _attend(A, b, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[:2] == 7).all()) and bool((out[-3:] == 7).all())
    want, wl, tol, ltol = R.attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], b["scale"])
    _close(out[2:-3], want[2:-3], tol[2:-3], "out")
    _close(lse[2:-3], wl[2:-3], ltol[2:-3], "lse")
    mass = torch.zeros((3, 2, b["table"].shape[1]), device="cuda")
    got = A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass, out=mass)
    want, tol = R.attention(b["q"], b["kp"], None, b["table"], b["lens"], b["starts"], b["scale"],
                            (lse, torch.zeros_like(mass), 1.0))
    assert got.data_ptr() == mass.data_ptr()
    _close(mass, want, tol, "mass in place")


def test_wrong_arrays_stay_in_bounds(A):
    """Lengths below 0 and behind the table, row starts that fall or leave q, a hint that is too small."""
    _say("wrong arrays")
    b = _batch([(3, 50), (4, 60), (9, 70)], 4, 2, 64, 16, BF, seed=6)
    for lens, starts in (([-5, 60, 2 ** 31 - 1], [0, 3, 7, 16]), ([50, 60, 70], [-3, 7, 2, 99]), ([0, 0, 0], [0, 3, 7, 16])):
        b["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        b["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        for most in (1, 100):
            b["most"] = most
            out, lse = _attend(A, b, out=torch.zeros_like(b["q"]))
            want, wl, tol, ltol = R.attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], b["scale"])
            rows = torch.zeros(16, dtype=torch.bool)
            for s in range(3):
                rows[max(starts[s], 0):max(starts[s + 1], 0)] = True
            if starts == [0, 3, 7, 16]:
                _close(out[rows.cuda()], want[rows], tol[rows], (lens, starts, most))
            A.attention_mass(b["q"], lse.nan_to_num(0, 0, 0), b["kp"], b["table"], b["lens"], b["starts"],
                             torch.zeros((3, 2, b["table"].shape[1]), device="cuda"))
    torch.cuda.synchronize()


def test_a_chunk_in_a_wide_table(A):
    """Pieces are cut by the sequences' lengths, not by the table's width: decoding sequences, one of them longer than
    the chunk's, beside two chunks; and the same chunk alone, whose pieces are others."""
    _say("wide table")
    for lens in ([(1, 40), (300, 3001), (1, 5000), (0, 7), (130, 131)], [(300, 3001)], [(40, 600), (33, 33)]):
        b = _batch(lens, 4, 2, 128, 16, BF, seed=11, extra_cols=3000)
        _, lse = _check_attend(A, b, lens)
        _check_mass(A, b, lse, lens)


@pytest.mark.parametrize("d", [64, 256])
def test_a_hint_too_small_by_many_rows(A, d):
    """Sequences whose rows come in many turns of a kernel made for 16: each turn begins with the last one's numbers
    read, so that every call gives the same bits."""
    _say("hint", d)
    b = _batch([(70, 200), (33, 33), (1, 90)], 5, 2, d, 16, BF, seed=8)
    b["most"] = 1
    first = _attend(A, b)
    for _ in range(8):
        again = _attend(A, b)
        assert all(torch.equal(x, y) for x, y in zip(first, again))
    want, wl, tol, ltol = R.attention(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b["starts"], b["scale"])
    _close(first[0], want, tol, "out")
    _close(first[1], wl, ltol, "lse")


def test_pages_beyond_32_bit_offsets(A):
    """A pool of more than 2^32 elements: the last pages are reached."""
    _say("large pool")
    pages, t, kv, d = 40000, 64, 8, 256   # 5.2e9 elements, 10.5 GB each
    kp = torch.empty((pages, t, kv, d), dtype=BF, device="cuda")
    vp = torch.empty((pages, t, kv, d), dtype=BF, device="cuda")
    ids = [pages - 1, 3, pages - 2, 33000]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in ids:
        kp[i] = torch.randn((t, kv, d), generator=gen, device="cuda").to(BF)
        vp[i] = torch.randn((t, kv, d), generator=gen, device="cuda").to(BF)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    small = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([250], dtype=torch.int32, device="cuda")
    for n in (1, 40):
        q = torch.randn((n, 16, d), generator=gen, device="cuda").to(BF)
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        a, la = A.paged_attention(q, kp, vp, table, lens, starts, return_lse=True)
        b, lb = A.paged_attention(q, kp[ids], vp[ids], small, lens, starts, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
        mass = torch.zeros((1, kv, 4), device="cuda")
        assert torch.equal(A.attention_mass(q, la, kp, table, lens, starts, mass),
                           A.attention_mass(q, la, kp[ids], small, lens, starts, mass))
    x = torch.randn((2, kv, d), generator=gen, device="cuda").to(BF)
    A.append_tokens(x, x, x, kp, vp, torch.tensor([pages * t - 1, 33000 * t], device="cuda"),
                    torch.zeros(2, dtype=torch.int32, device="cuda"), A.rope_table(1, 0))
    assert torch.equal(kp[-1, -1], x[0]) and torch.equal(vp[33000, 0], x[1])


def test_nothing_to_do(A):
    b = _batch([(1, 5), (2, 9)], 2, 1, 64, 16, BF)
    none = torch.zeros((0, 2, 64), dtype=BF, device="cuda")
    out, lse = A.paged_attention(none, b["kp"], b["vp"], b["table"], b["lens"], torch.zeros(3, dtype=torch.int32, device="cuda"),
                                 return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    mass = torch.ones((2, 1, 1), device="cuda")
    got = A.attention_mass(none, lse, b["kp"], b["table"], b["lens"], torch.zeros(3, dtype=torch.int32, device="cuda"), mass,
                           decay=0.25)
    assert bool((got == 0.25).all())
    no = lambda x: x[:0].contiguous()  # noqa: E731
    out = A.paged_attention(none, b["kp"], b["vp"], no(b["table"]), no(b["lens"]), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 2, 64)
    e = A.evict_pages(no(mass), no(b["table"]), no(b["lens"]), page_tokens=16, budget=1)
    assert e.page_table.shape == (0, 1)


# ---- eviction ----------------------------------------------------------------------

@pytest.mark.parametrize("s,heads,mp,t", [(1, 1, 1, 16), (3, 8, 64, 16), (5, 3, 1000, 13), (2, 9, 1025, 1), (4, 2, 4100, 16),
                                          (1, 1, 20000, 64), (2, 17, 300, 7)])
def test_evict(A, s, heads, mp, t):
    _say("evict", s, heads, mp, t)
    gen = torch.Generator().manual_seed(mp)
    for trial, (budget, sink, recent) in enumerate([(mp // 2, 1, 1), (0, 0, 1), (3, 4, 2), (mp, 0, 1), (mp // 3, 0, mp + 5),
                                                    (max(mp - 1, 0), 2, 1), (mp // 4, mp + 1, 1)]):
        mass = torch.exp(4 * torch.randn((s, heads, mp), generator=gen))
        if trial % 3 == 1:   # many equal ones, both zeros, infinities, NaN
            mass = torch.randint(0, 3, (s, heads, mp), generator=gen).float() * torch.tensor([1.0, -0.0])[
                torch.randint(0, 2, (s, heads, mp), generator=gen)]
            mass[:, 0, ::7] = math.inf
            mass[:, 0, ::11] = math.nan
            mass[:, 0, ::13] = -math.inf
        lens = torch.randint(0, mp * t + 1, (s,), generator=gen).int()
        lens[0] = mp * t
        table = torch.randint(-1, 10000, (s, mp), generator=gen).int()
        want = R.evict(mass, table, lens, t, budget, sink, recent)
        args = dict(page_tokens=t, budget=budget, sink=sink, recent=recent)
        m, tb, ln = mass.cuda(), table.cuda(), lens.cuda()
        got = A.evict_pages(m, tb, ln, **args)
        for name, g, w in zip(got._fields, got, want):
            assert torch.equal(g.cpu().nan_to_num(-5.5) if g.is_floating_point() else g.cpu(),
                               w.nan_to_num(-5.5) if w.is_floating_point() else w), (trial, name)
        assert torch.equal(tb.cpu(), table)
        again = A.evict_pages(m, tb, ln, in_place=True, **args)
        assert again.mass.data_ptr() == m.data_ptr()
        for name, g, w in zip(got._fields, again, got):
            assert torch.equal(g.nan_to_num(-5.5) if g.is_floating_point() else g,
                               w.nan_to_num(-5.5) if w.is_floating_point() else w), (trial, name, "in place")


def test_evict_wrong_lengths(A):
    _say("evict, wrong lengths")
    mass = torch.rand((2, 2, 8), device="cuda")
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    e = A.evict_pages(mass, table, torch.tensor([-4, 10 ** 6], dtype=torch.int32, device="cuda"), page_tokens=16, budget=5)
    assert e.n_evicted.tolist() == [0, 3] and e.kv_lens.tolist() == [-4, 10 ** 6 - 48]
    assert bool((e.page_table[0] == -1).all())


# ---- together, streams, graphs -------------------------------------------------------

def test_a_serving_run(A):
    """Prompts enter their pages, decode, keep their accounts, give up pages, which go cold, come back into other pages and
    are attended to again."""
    import vlx_tee_amd.pages as PG
    import vlx_tee_amd.workloads as W
    _say("serving run")
    t, kv, g, d, r, pages, s = 16, 2, 4, 128, 64, 64, 3
    gen = torch.Generator(device="cuda").manual_seed(3)
    kp = torch.zeros((pages, t, kv, d), dtype=BF, device="cuda")
    vp = torch.zeros_like(kp)
    rope = A.rope_table(4096, r)
    w = (torch.ones(d, device="cuda")).to(BF)
    table = torch.arange(s * 16, dtype=torch.int32, device="cuda").view(s, 16).contiguous()
    mass = torch.zeros((s, kv, 16), device="cuda")
    lens = torch.zeros(s, dtype=torch.int32, device="cuda")
    positions = [0] * s

    def step(counts):
        nonlocal lens, mass
        n = sum(counts)
        x = torch.randn((n, g * kv + 2 * kv, d), generator=gen, device="cuda").to(BF)
        have = lens.tolist()
        slots, pos = [], []
        for i, c in enumerate(counts):
            for j in range(c):
                slots.append(int(table[i, (have[i] + j) // t]) * t + (have[i] + j) % t)
                pos.append(positions[i] + j)
            positions[i] += c
        q = A.append_tokens(x[:, :g * kv], x[:, g * kv:g * kv + kv], x[:, g * kv + kv:], kp, vp,
                            torch.tensor(slots, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda"), rope,
                            q_weight=w, k_weight=w)
        lens += torch.tensor(counts, dtype=torch.int32, device="cuda")
        starts = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device="cuda")
        out, lse = A.paged_attention(q, kp, vp, table, lens, starts, return_lse=True, max_q_len=max(counts))
        want, wl, tol, ltol = R.attention(q, kp, vp, table, lens, starts, d ** -0.5)
        _close(out, want, tol, counts)
        _close(lse, wl, ltol, counts)
        before = mass.clone()
        A.attention_mass(q, lse, kp, table, lens, starts, mass, out=mass)
        want, tol = R.attention(q, kp, None, table, lens, starts, d ** -0.5, (lse, before, 1.0))
        _close(mass, want, tol, counts)
        return float(lens.sum())

    step([180, 77, 33])
    for _ in range(3):
        step([1, 1, 1])
    total = mass.sum(2)   # each of a KV head's 4 query heads gave weight 1 a token
    assert torch.allclose(total[:, 0].cpu(), torch.tensor([183.0, 80.0, 36.0]) * 4, rtol=1e-4)
    e = A.evict_pages(mass, table, lens, page_tokens=t, budget=6, sink=1, recent=2)
    assert e.n_evicted.tolist() == [6, 0, 0]
    gone = e.evicted[0, :6].long()
    # those pages go cold and come back into pages of their own
    blob = 48 + W.WORKLOADS["c2_k8v4_prefix1g"].geometry.payload_bytes(3, 2)
    geo = dict(num_tokens=t, num_heads=kv, head_dim=d, rope_dim=r, dtype=BF, is_mla_single_buffer=False)
    import vlx_tee_amd.spec as spec
    payload = spec.ColdPageGeometry(t, kv, d, r).payload_bytes(3, 2)
    blobs = torch.zeros((pages, 48 + payload), dtype=torch.uint8, device="cuda")
    idx = np.arange(pages)
    descs = PG.build_descriptors(kp, vp, blobs, idx, idx.astype(np.uint64), np.zeros(pages))
    keys = W.session_keys()
    PG.egress(descs[gone].contiguous(), 6, preset=3, rope_mode=2, expected_payload_bytes=payload, tenant_id_hash=1,
              model_id_hash=2, **geo, **keys)
    old = kp[gone].clone()
    kp[gone] = 0
    k2, v2 = torch.zeros_like(kp), torch.zeros_like(vp)
    back = PG.build_descriptors(k2, v2, blobs, idx, idx.astype(np.uint64), np.zeros(pages))
    assert PG.ingress(back[gone].contiguous(), 6, 48 + payload, expected_tenant_hash=1, expected_model_hash=2, **geo, **keys) == 0
    assert float((k2[gone].float() - old.float()).abs().max()) < 0.1 * float(old.float().abs().max())
    table, mass, lens = e.page_table, e.mass, e.kv_lens
    step([1, 1, 1])
    full = torch.cat([table[:1, :6], gone[None].int()], 1)   # the cold pages in front of nothing: attended once more
    kp[gone], vp[gone] = k2[gone], v2[gone]
    table = torch.cat([full, torch.full((1, 4), -1, dtype=torch.int32, device="cuda")], 1).repeat(s, 1).contiguous()
    del blob
    q = torch.randn((s, g * kv, d), generator=gen, device="cuda").to(BF)
    lens = torch.full((s,), 12 * t, dtype=torch.int32, device="cuda")
    starts = torch.arange(s + 1, dtype=torch.int32, device="cuda")
    out = A.paged_attention(q, kp, vp, table, lens, starts)
    want, _, tol, _ = R.attention(q, kp, vp, table, lens, starts, d ** -0.5)
    _close(out, want, tol, "after ingress")


def test_two_calls_at_once_on_two_streams(A):
    _say("two streams")
    bs = [_batch([(1, 3000), (40, 900)], 4, 2, 128, 16, BF, seed=i) for i in range(2)]
    want = [_attend(A, b) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, b in enumerate(bs):
            with torch.cuda.stream(streams[i]):
                got[i].append(_attend(A, b))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_the_same_call_gives_the_same_bits(A):
    _say("same bits")
    b = _batch([(1, 3000), (200, 900), (1, 77)], 4, 2, 128, 16, BF, seed=1)
    out, lse = _attend(A, b)
    mass = torch.zeros((3, 2, b["table"].shape[1]), device="cuda")
    m = A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass)
    for _ in range(5):
        o2, l2 = _attend(A, b)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        assert torch.equal(m, A.attention_mass(b["q"], lse, b["kp"], b["table"], b["lens"], b["starts"], mass))


def test_captured_steps(A):
    """Two graphs of a decoding step, captured over one batch's arrays, replayed in turn as the arrays change, beside eager
    calls."""
    _say("graphs")
    b = _batch([(1, 700), (1, 90), (1, 2000)], 4, 2, 128, 16, BF, seed=8)
    mass = torch.zeros((3, 2, b["table"].shape[1]), device="cuda")
    x = torch.randn((3, 12, 128), device="cuda").to(BF)
    slots = torch.tensor([5, 6, 7], device="cuda")
    pos = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    rope = A.rope_table(64, 64)

    def step():
        q = A.append_tokens(x[:, :8], x[:, 8:10], x[:, 10:], b["kp"], b["vp"], slots, pos, rope)
        out, lse = A.paged_attention(q, b["kp"], b["vp"], b["table"], b["lens"], b["starts"], max_q_len=1, return_lse=True)
        m = A.attention_mass(q, lse, b["kp"], b["table"], b["lens"], b["starts"], mass)
        return [out, lse, m, *A.evict_pages(m, b["table"], b["lens"], page_tokens=16, budget=20)]

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(6):
        x.normal_()
        pos.fill_(i)
        b["lens"].copy_(torch.tensor([700 - i, 3 * i, 1000 + 100 * i], dtype=torch.int32))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph, outs = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(outs, want):
            assert torch.equal(a, w), i
