"""Arguments that allot_pages and release_pages refuse, through the C ABI (its checks come before any use of the GPU, so the
addresses here are never read) and the Python module.  No GPU needed."""
from __future__ import annotations

import pytest
import torch

from test_hot_refusals import N  # noqa: F401  (the module's fixture)

B = 0x10000000


def _allot(N, **kw):
    a = dict(table=B, stride=8, cols=8, lens=B + 0x10000, wanted=B + 0x20000, s=4, free=B + 0x30000, cap=100,
             n_free=B + 0x40000, counts=None, t=16, rows=64, ol=B + 0x50000, on=B + 0x60000, oc=None, starts=B + 0x70000,
             slots=B + 0x80000, pos=B + 0x90000, granted=B + 0xA0000, work=B + 0xB0000, bytes=1 << 20)
    a.update(kw)
    rc = N.lib().ztcp_allot_pages(a["table"], a["stride"], a["cols"], a["lens"], a["wanted"], a["s"], a["free"], a["cap"],
                                  a["n_free"], a["counts"], a["t"], a["rows"], a["ol"], a["on"], a["oc"], a["starts"],
                                  a["slots"], a["pos"], a["granted"], a["work"], a["bytes"], None)
    return rc, N.last_error()


def _release(N, **kw):
    a = dict(table=B, stride=8, cols=8, lens=B + 0x10000, s=4, t=16, free=B + 0x30000, cap=100, n_free=B + 0x40000,
             ot=B + 0x50000, ots=8, on=B + 0x60000, released=B + 0x70000, work=B + 0xB0000, bytes=1 << 20)
    a.update(kw)
    rc = N.lib().ztcp_release_pages(a["table"], a["stride"], a["cols"], a["lens"], a["s"], a["t"], a["free"], a["cap"],
                                    a["n_free"], a["ot"], a["ots"], a["on"], a["released"], a["work"], a["bytes"], None)
    return rc, N.last_error()


COMMON = [(dict(s=-1), "n_seqs"), (dict(s=1 << 24), "n_seqs"), (dict(t=0), "num_tokens"), (dict(cols=0), "num_tokens"),
          (dict(t=1 << 31), "num_tokens"), (dict(cols=1 << 27), "below 2^31"), (dict(stride=7), "cover"),
          (dict(table=None), "page_table"), (dict(cap=-1), "capacity"), (dict(cap=1 << 31), "capacity"), (dict(lens=None), "NULL"),
          (dict(n_free=None), "NULL"), (dict(free=None), "NULL"), (dict(on=None), "NULL")]
WORK = [(dict(work=None), "workspace"), (dict(work=B + 0xB0002), "workspace"), (dict(bytes=16), "workspace")]


@pytest.mark.parametrize("kw,why", COMMON + [
    (dict(rows=-1), "max_rows"), (dict(rows=(1 << 31) - 1024), "max_rows"), (dict(counts=B + 0xC0000), "both"),
    (dict(oc=B + 0xC0000), "both"), (dict(wanted=None), "NULL"), (dict(ol=None), "NULL"), (dict(starts=None), "NULL"),
    (dict(slots=None), "NULL"), (dict(pos=None), "NULL"), (dict(granted=None), "NULL")]
    + [(dict(kw, rows=5000), why) for kw, why in WORK])
def test_allot_arguments(N, kw, why):
    rc, msg = _allot(N, **kw)
    assert rc == N.EINVAL and why in msg, msg


@pytest.mark.parametrize("kw,why", COMMON + WORK + [(dict(ots=7), "cover"), (dict(ot=None), "NULL"), (dict(released=None), "NULL")])
def test_release_arguments(N, kw, why):
    rc, msg = _release(N, **kw)
    assert rc == N.EINVAL and why in msg, msg


def test_overlaps(N):
    for kw in (dict(ol=B + 0x20000), dict(ol=B + 0x10004), dict(on=B + 0x10000), dict(starts=B + 4), dict(slots=B + 0x30000),
               dict(pos=B + 0x80008), dict(granted=B + 0x50000), dict(work=B + 0x70000, rows=5000), dict(free=B + 16), dict(lens=B),
               dict(counts=B + 0xC0000, oc=B + 0xC0004)):
        assert _allot(N, **kw)[0] == N.EOVERLAP, kw
    for kw in (dict(ot=B + 4), dict(ot=B, ots=16), dict(on=B), dict(released=B + 0x10000), dict(free=B + 8), dict(work=B + 0x30000),
               dict(released=B + 0x60000), dict(ot=B + 0x30000)):
        assert _release(N, **kw)[0] == N.EOVERLAP, kw


def test_workspaces(N):
    L, bad = N.lib(), (1 << 64) - 1
    assert L.ztcp_allot_pages_workspace(0, 0) == 0 and L.ztcp_allot_pages_workspace(2000, 10) >= 16 * 2000
    for args in ((-1, 1), (1 << 24, 1), (1, -1), (1, (1 << 31) - 1024)):
        assert L.ztcp_allot_pages_workspace(*args) == bad
    assert L.ztcp_release_pages_workspace(3, 10) >= 8 * 4
    for args in ((-1, 1), (1 << 24, 1), (1, 0), (1, 1 << 31)):
        assert L.ztcp_release_pages_workspace(*args) == bad


def test_python_checks(N):
    import vlx_tee_amd.attention as A

    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="page_table must be a HIP tensor"):
        A.allot_pages(i32[None], i32, i32, i32, i32, page_tokens=16, max_rows=1)
    with pytest.raises(ValueError, match="page_table must be a HIP tensor"):
        A.release_pages(i32[None], i32, i32, i32, page_tokens=16)
    with pytest.raises(ValueError, match="q_lens must be a tensor"):
        A.allot_pages(i32[None], i32, 1, i32, i32, page_tokens=16, max_rows=1)
    with pytest.raises(ValueError, match="max_rows must be a whole number"):
        A.allot_pages(i32[None], i32, i32, i32, i32, page_tokens=16, max_rows=1 << 70)
