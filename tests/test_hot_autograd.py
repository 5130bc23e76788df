"""What the operators on hot pages, which have no derivatives, do with tensors that carry one.  No GPU needed: these checks
come before those of the devices."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD


@pytest.fixture(scope="module")
def A(pkg):
    import vlx_tee_amd.attention as A

    return A


def _calls(A):
    """(name of an argument, a call that passes it)"""
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    pages = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    mass, rope, w = torch.zeros((1, 2, 1)), torch.zeros((4, 64)), torch.ones(64, dtype=torch.bfloat16)
    attend = lambda q=x, k=pages, v=pages: A.paged_attention(q, k, v, i32[None], i32[:1], i32)  # noqa: E731
    append = lambda k=x[:, :2], r=rope, w=w: A.append_tokens(x, k, x[:, :2], pages, pages, i32.long(), i32, r,  # noqa: E731
                                                             q_weight=w)
    yield "q", x, lambda t: attend(q=t)
    yield "k_pages", pages, lambda t: attend(k=t)
    yield "v_pages", pages, lambda t: attend(v=t)
    yield "k", x[:, :2], lambda t: append(k=t)
    yield "rope", rope, lambda t: append(r=t)
    yield "q_weight", w, lambda t: append(w=t)
    yield "lse", torch.zeros((2, 4)), lambda t: A.attention_mass(x, t, pages, i32[None], i32[:1], i32, mass)
    yield "mass", mass, lambda t: A.attention_mass(x, torch.zeros((2, 4)), pages, i32[None], i32[:1], i32, t)
    yield "mass", mass, lambda t: A.evict_pages(t, i32[None], i32[:1], page_tokens=16, budget=1)


def test_a_forward_tangent_is_refused(A):
    """It would be dropped without a word; torch.no_grad() does not switch tangents off."""
    for name, t, call in _calls(A):
        with fwAD.dual_level():
            dual = fwAD.make_dual(t, torch.ones_like(t))
            with pytest.raises(ValueError, match=f"{name} carries a tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match=f"{name} carries a tangent"):
                call(dual)
            with fwAD._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="HIP"):   # on the CPU; not the tangent
                call(dual)


def test_a_gradient_is_refused_with_grad_mode_on(A):
    for name, t, call in _calls(A):
        t = t.clone().requires_grad_()
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call(t)
        with torch.no_grad(), pytest.raises(ValueError, match="HIP"):
            call(t)
