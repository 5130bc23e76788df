"""Arguments that the operators on hot pages refuse, through the C ABI (its checks come before any use of the GPU, so
the addresses here are never read) and the Python module.  No GPU needed."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

K, V, Q, O, W = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def N(pkg):
    import vlx_tee_amd._native as N

    return N


def _geo(N, t=16, h=2, d=128, r=64, dt=1):
    return N.geometry(t, h, d, r, dt, False)


def _pool(N, **kw):
    a = dict(k=K, v=V, n_pages=8, k_stride=4096, v_stride=4096)
    a.update(kw)
    return N.PagePool(**a)


def _append(N, geo=None, pool=None, **kw):
    a = dict(q=Q, qs=1024, qo=O, qos=1024, k=W, ks=256, v=W + 0x100000, vs=256, n=4, heads=8, slots=Q + 0x800000,
             pos=Q + 0x900000, rope=Q + 0xA00000, maxpos=100, qw=None, qwl=0, kw=None, kwl=0, eps=1e-6, inter=0)
    a.update(kw)
    geo, pool = geo or _geo(N), pool or _pool(N)
    rc = N.lib().ztcp_append_tokens(a["q"], a["qs"], a["qo"], a["qos"], a["k"], a["ks"], a["v"], a["vs"], a["n"],
                                    a["heads"], C.byref(pool), C.byref(geo), a["slots"], a["pos"], a["rope"], a["maxpos"],
                                    a["qw"], a["qwl"], a["kw"], a["kwl"], a["eps"], a["inter"], None)
    return rc, N.last_error()


BAD_GEO = [dict(t=0), dict(h=0), dict(d=8), dict(d=24), dict(r=8), dict(r=-16), dict(r=144), dict(dt=2),
           dict(t=1 << 20, h=1 << 10)]
BAD_POOL = [dict(n_pages=0), dict(n_pages=1 << 31), dict(k=None), dict(k=K + 8), dict(v=V + 2), dict(k_stride=4088),
            dict(v_stride=4000), dict(k_stride=4100)]


@pytest.mark.parametrize("geo", BAD_GEO)
def test_geometry(N, geo):
    assert _append(N, geo=_geo(N, **geo))[0] == N.EINVAL
    assert _attend(N, geo=_geo(N, **geo))[0] == N.EINVAL
    assert _mass(N, geo=_geo(N, **geo))[0] == N.EINVAL


@pytest.mark.parametrize("pool", BAD_POOL)
def test_pool(N, pool):
    assert _append(N, pool=_pool(N, **pool))[0] == N.EINVAL
    assert _attend(N, pool=_pool(N, **pool))[0] == N.EINVAL
    if "v" not in pool:
        assert _mass(N, pool=_pool(N, **pool))[0] == N.EINVAL


@pytest.mark.parametrize("kw,why", [
    (dict(n=-1), "negative"), (dict(heads=-1), "negative"), (dict(n=1 << 31), "too many"), (dict(k=None), "NULL"),
    (dict(q=None), "NULL"), (dict(qo=None), "NULL"), (dict(slots=None), "NULL"), (dict(pos=None), "NULL"),
    (dict(rope=None), "NULL"), (dict(v=None), "both"), (dict(maxpos=0), "max_position"), (dict(maxpos=1 << 31), "max_position"),
    (dict(qw=W, qwl=100), "entries"), (dict(kw=W, kwl=-64), "entries"), (dict(qw=W), "agree"), (dict(kwl=128), "agree"),
    (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps"), (dict(eps=INF), "eps"), (dict(q=Q + 2), "aligned"),
    (dict(ks=257), "aligned"), (dict(qw=W + 2, qwl=128), "aligned"), (dict(qs=1000), "cover"), (dict(vs=128), "cover")])
def test_append_arguments(N, kw, why):
    rc, msg = _append(N, **kw)
    assert rc == N.EINVAL and why in msg, msg


def test_append_overlaps(N):
    base = 0x70000000
    for kw in (dict(qo=Q + 16), dict(qo=W), dict(k=O), dict(k=K + 32, ks=256), dict(v=V + 8 * 8192 - 16), dict(qo=K),
               dict(qo=Q, qos=2048)):
        assert _append(N, **kw)[0] == N.EOVERLAP, kw
    assert _append(N, pool=_pool(N, v=K + 16))[0] == N.EOVERLAP
    # views side by side in one buffer do not overlap, one that reaches into its neighbour does
    row = (8 + 2 + 2) * 128
    side = dict(q=base, qs=row, k=base + 2 * 1024, ks=row, v=base + 2 * 1280, vs=row)
    assert _append(N, **side, qo=base + 2 * 64, qos=row)[0] == N.EOVERLAP
    assert _append(N, **side, qo=base + 2 * row * 8 - 512, qos=row, n=4)[0] != N.EINVAL
    assert _append(N, n=0)[0] == N.OK


def _batch(N, **kw):
    a = dict(page_table=Q + 0x800000, table_stride=4, max_pages=4, kv_lens=Q + 0x900000, q_starts=Q + 0xA00000, n_seqs=2,
             n_rows=2, max_q_len=1)
    a.update(kw)
    return N.PagedBatch(**a)


def _attend(N, geo=None, pool=None, batch=None, **kw):
    a = dict(q=Q, qs=1024, out=O, lse=None, heads=8, scale=0.1, work=W, bytes=1 << 30)
    a.update(kw)
    geo, pool, batch = geo or _geo(N), pool or _pool(N), batch or _batch(N)
    rc = N.lib().ztcp_paged_attention(a["q"], a["qs"], a["out"], a["lse"], a["heads"], C.byref(pool), C.byref(batch),
                                      C.byref(geo), a["scale"], a["work"], a["bytes"], None)
    return rc, N.last_error()


def _mass(N, geo=None, pool=None, batch=None, **kw):
    a = dict(q=Q, qs=1024, lse=W, heads=8, scale=0.1, mass=O, decay=1.0, out=O)
    a.update(kw)
    geo, pool, batch = geo or _geo(N), pool or _pool(N), batch or _batch(N)
    rc = N.lib().ztcp_attention_mass(a["q"], a["qs"], a["lse"], a["heads"], C.byref(pool), C.byref(batch), C.byref(geo),
                                     a["scale"], a["mass"], a["decay"], a["out"], None)
    return rc, N.last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=-1), dict(n_seqs=1 << 24), dict(n_rows=-1), dict(n_rows=1 << 31),
                                dict(max_q_len=-1), dict(max_pages=0), dict(max_pages=1 << 28), dict(page_table=None),
                                dict(kv_lens=None), dict(q_starts=None), dict(table_stride=3), dict(n_rows=1 << 28)])
def test_batch(N, kw):
    assert _attend(N, batch=_batch(N, **kw))[0] == N.EINVAL
    assert _mass(N, batch=_batch(N, **kw))[0] == N.EINVAL
    geo, pool, batch = _geo(N), _pool(N), _batch(N, **kw)
    assert N.lib().ztcp_paged_attention_workspace(C.byref(batch), C.byref(pool), C.byref(geo), 8) == C.c_size_t(-1).value


@pytest.mark.parametrize("kw", [dict(heads=0), dict(heads=7), dict(heads=1 << 17), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=NAN), dict(scale=INF), dict(q=None), dict(q=Q + 8), dict(qs=1020), dict(qs=512)])
def test_attention_and_mass_arguments(N, kw):
    assert _attend(N, **kw)[0] == N.EINVAL
    assert _mass(N, **kw)[0] == N.EINVAL


def test_attention_needs_both_buffers_and_widths_up_to_256(N):
    assert _attend(N, pool=_pool(N, v=None))[0] == N.EINVAL
    wide = dict(geo=_geo(N, d=272, r=0), pool=_pool(N, k_stride=16 * 2 * 272, v_stride=16 * 2 * 272))
    assert _attend(N, **wide) == (N.EINVAL, "head_dim must be at most 256")
    assert _mass(N, **wide)[0] == N.EINVAL
    assert _attend(N, out=None)[0] == N.EINVAL and _attend(N, out=O + 4)[0] == N.EINVAL


def test_mass_arguments(N):
    for kw in (dict(mass=None), dict(out=None), dict(lse=None), dict(decay=-0.5), dict(decay=NAN), dict(decay=INF)):
        assert _mass(N, **kw)[0] == N.EINVAL, kw
    for kw in (dict(out=O + 4), dict(out=Q), dict(out=W), dict(out=K + 64)):
        assert _mass(N, **kw)[0] == N.EOVERLAP, kw
    assert _mass(N, batch=_batch(N, n_seqs=0))[0] == N.OK


def _evict(N, **kw):
    a = dict(mass=Q, table=K, stride=8, lens=V, s=2, heads=2, mp=8, t=16, budget=4, sink=1, recent=1, ot=O, ots=8,
             om=O + 0x1000, ol=O + 0x2000, ev=O + 0x3000, ne=O + 0x4000)
    a.update(kw)
    rc = N.lib().ztcp_evict_pages(a["mass"], a["table"], a["stride"], a["lens"], a["s"], a["heads"], a["mp"], a["t"],
                                  a["budget"], a["sink"], a["recent"], a["ot"], a["ots"], a["om"], a["ol"], a["ev"], a["ne"],
                                  None)
    return rc


def test_evict_arguments(N):
    for kw in (dict(s=-1), dict(heads=0), dict(mp=0), dict(t=0), dict(mp=1 << 27), dict(mp=(1 << 31) - 4095, t=1),
               dict(budget=-1), dict(sink=-1),
               dict(recent=0), dict(stride=7), dict(ots=7), dict(mass=None), dict(table=None), dict(lens=None),
               dict(ot=None), dict(om=None), dict(ol=None), dict(ev=None), dict(ne=None)):
        assert _evict(N, **kw) == N.EINVAL, kw
    for kw in (dict(ev=K), dict(ev=Q + 16), dict(ot=K + 4), dict(ot=K, ots=16), dict(om=Q + 4), dict(ol=K), dict(ne=V),
               dict(ev=O), dict(ne=O + 0x3000 + 8)):
        assert _evict(N, **kw) == N.EOVERLAP, kw
    assert _evict(N, s=0) == N.OK


def test_python_checks(N):
    import vlx_tee_amd.attention as A

    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    pages = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP float16 or bfloat16"):
        A.paged_attention(x, pages, pages, i32[None], i32[:1], i32)
    with pytest.raises(ValueError, match="HIP float16 or bfloat16"):
        A.append_tokens(x, x[:, :2], x[:, :2], pages, pages, i32.long(), i32, torch.zeros((4, 64)))
    with pytest.raises(ValueError, match="single-buffer"):
        A.paged_attention(x, pages, None, i32[None], i32[:1], i32)
    with pytest.raises(ValueError, match="mass must be a HIP tensor"):
        A.evict_pages(torch.zeros((1, 2, 2)), i32[None], i32[:1], page_tokens=16, budget=1)
    with pytest.raises(ValueError, match="k_pages requires a gradient"):
        A.paged_attention(x, pages.clone().requires_grad_(), pages, i32[None], i32[:1], i32)
    with pytest.raises(ValueError, match="q must be a tensor"):
        A.paged_attention(None, pages, pages, i32[None], i32[:1], i32)
    with pytest.raises(ValueError, match="return_lse must be true or false"):
        A.paged_attention(x, pages, pages, i32[None], i32[:1], i32, return_lse=torch.ones(2))
    with pytest.raises(ValueError, match="even"):
        A.rope_table(4, 3, device="cpu")
    t = A.rope_table(9, 4, base=100.0, device="cpu")
    assert torch.allclose(t[8], torch.tensor([8.0, 0.8]).repeat(2).double().cos().float() * torch.tensor([1, 1, 0, 0])
                          + torch.tensor([8.0, 0.8]).repeat(2).double().sin().float() * torch.tensor([0, 0, 1, 1]))
