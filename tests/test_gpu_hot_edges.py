"""GPU tests of the operators on hot pages at the edges of their ranges: the largest sizes, numbers that are not finite
in every place of a tile, and what torch keeps of tensors that are written in place."""
from __future__ import annotations

import pytest
import torch

import hot_reference as R
from test_gpu_hot_ops import A, BF, _close, _say  # noqa: F401  (A: the module's fixture)

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
