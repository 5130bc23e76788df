"""GPU tests of the operators on hot pages at the edges of their ranges: the largest sizes, numbers that are not finite
in every place of a tile, and what torch keeps of tensors that are written in place."""
from __future__ import annotations

import pytest
import torch

import hot_reference as R
from test_gpu_hot_ops import A, BF, FP, _batch, _check_attend, _close, _say  # noqa: F401  (A: the module's fixture)

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
