"""Operators on hot KV pages: the steps of a serving engine around the codec.

A step's new tokens enter their pages (``append_tokens``: norms of queries and
keys, position rotation and the write in one pass), attend over their
sequences' pages (``paged_attention``), and add to the account of every page
the attention weight it received (``attention_mass``).  A sequence with more
pages than its budget gives up those with the least weight (``evict_pages``);
their ids select the descriptors that ``pages.egress`` takes to the cold tier,
and pages that ``pages.ingress`` brought back are read like any other.

Pages are the codec's hot pages: a pool ``[n_pages, page_tokens, kv_heads,
head_dim]`` of float16 or bfloat16, each page contiguous (pages may be padded
or interleaved), RoPE columns leading.  Row ``s`` of ``page_table`` lists
sequence ``s``'s pages in order; an entry outside the pool is a page that is
not there (cold) and takes no part.  ``kv_lens`` counts a sequence's tokens,
the new ones among them, which are rows ``q_starts[s]`` to ``q_starts[s + 1]``
of ``q``.

Every call is enqueued on the current stream of its tensors' device,
synchronizes nothing, and can be recorded into a graph.  No operator has a
gradient: they serve, as the codec does.  Wrong arguments raise
``ValueError``; indexes on the device are bounded by the kernels as
include/ztcp.h says (ztcp_append_tokens and the entries after it).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _native as N

_DTYPES = {torch.float16: N.HOT_FP16, torch.bfloat16: N.HOT_BF16}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _raise(rc: int, what: str) -> None:
    if rc in (N.EINVAL, N.EOVERLAP):
        raise ValueError(f"{what}: {N.last_error()}")
    if rc != N.OK:
        raise RuntimeError(f"{what}: {N.strerror(rc)} (code {rc})")


def _stream(device: torch.device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _tokens(t: torch.Tensor, name: str, like: torch.Tensor, heads: int | None = None) -> int:
    """Elements between the tokens of [tokens, heads, head_dim] rows."""
    _check(isinstance(t, torch.Tensor) and t.dim() == 3, f"{name} must have shape [tokens, heads, head_dim]")
    _check(t.dtype == like.dtype and t.device == like.device, f"{name} must match the pages' dtype and device")
    _check(t.size(2) == like.size(3), f"{name}'s head_dim must be the pages'")
    _check(heads is None or t.size(1) == heads, f"{name} must have the pages' heads")
    # a dimension of one element may report any stride
    _check((t.size(2) == 1 or t.stride(2) == 1) and (t.size(1) <= 1 or t.stride(1) == t.size(2)),
           f"a token's heads must be contiguous in {name}")
    return t.stride(0) if t.size(0) > 1 else t.size(1) * t.size(2)


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor | None) -> N.PagePool:
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t is None:
            continue
        _check(isinstance(t, torch.Tensor) and t.dim() == 4,
               f"{name} must have shape [n_pages, page_tokens, kv_heads, head_dim]")
        _check(t.is_cuda and t.dtype in _DTYPES, f"{name} must be a HIP float16 or bfloat16 tensor")
        _check(t.size(0) > 0 and t[0].is_contiguous(), f"{name} must hold pages, each of them contiguous")
        _check(t.shape == k_pages.shape and t.dtype == k_pages.dtype and t.device == k_pages.device,
               "v_pages must match k_pages in shape, dtype and device")
    step = lambda t: t.stride(0) if t.size(0) > 1 else t[0].numel()  # noqa: E731
    return N.PagePool(k_pages.data_ptr(), None if v_pages is None else v_pages.data_ptr(), k_pages.size(0),
                      step(k_pages), step(k_pages if v_pages is None else v_pages))


def _array(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> int:
    _check(isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == device and t.is_contiguous()
           and tuple(t.shape) == shape, f"{name} must be a contiguous {str(dtype)[6:]} tensor of shape {list(shape)} "
           "on the pages' device")
    return t.data_ptr()


def _table(t: torch.Tensor, name: str, device: torch.device) -> int:
    """Entries between the rows of a page table."""
    _check(isinstance(t, torch.Tensor) and t.dim() == 2 and t.dtype == torch.int32 and t.device == device
           and t.size(1) > 0 and (t.size(1) == 1 or t.stride(1) == 1),
           f"{name} must be an int32 tensor [sequences, pages] on the pages' device, its rows contiguous")
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _batch(page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, n_rows: int,
           max_q_len: int | None, device: torch.device) -> N.PagedBatch:
    stride = _table(page_table, "page_table", device)
    s, mp = page_table.shape
    _check(max_q_len is None or max_q_len >= 0, "max_q_len must not be negative")
    return N.PagedBatch(page_table.data_ptr(), stride, mp, _array(kv_lens, "kv_lens", torch.int32, (s,), device),
                        _array(q_starts, "q_starts", torch.int32, (s + 1,), device), s, n_rows, max_q_len or 0)


def _geometry(k_pages: torch.Tensor, rope_dim: int, single: bool) -> N.Geometry:
    return N.geometry(k_pages.size(1), k_pages.size(2), k_pages.size(3), rope_dim, _DTYPES[k_pages.dtype], single)


def rope_table(max_position: int, rope_dim: int, base: float = 10000.0,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """[max_position, rope_dim] float32: the cosines, then the sines, of each
    position's rope_dim / 2 angles ``position * base ** (-2 i / rope_dim)``.
    The angles are computed in 64 bits: at position 100,000 a 32-bit angle is
    off by up to 2^-8."""
    _check(max_position > 0 and rope_dim >= 0 and rope_dim % 2 == 0, "max_position must be positive, rope_dim even")
    i = torch.arange(0, rope_dim, 2, dtype=torch.float64, device=device)
    a = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * base ** (-i / max(rope_dim, 1))
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def append_tokens(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, k_pages: torch.Tensor,
                  v_pages: torch.Tensor | None, slots: torch.Tensor, positions: torch.Tensor, rope: torch.Tensor, *,
                  q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  interleaved: bool = False, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Norms and rotates ``q`` and ``k`` and writes ``k`` and ``v`` into their
    pages; returns the queries (``q_out`` if given; it may be ``q`` itself).

    ``q`` [n, q_heads, d], ``k`` and ``v`` [n, kv_heads, d] may be views of one
    projection's output.  ``slots`` (int64) is page * page_tokens + token of
    each new token; one outside the pool writes no page.  ``rope`` is a
    ``rope_table``; its width is the number of rotated leading columns, paired
    half a width apart or, ``interleaved``, with their neighbours; row
    ``positions[i]`` (int32) holds token i's angles.  A weight of d entries
    norms each head vector, one of d - rope_dim entries the columns behind
    the rotated ones (the latent of single-buffer pages, whose ``v`` and
    ``v_pages`` are None), None nothing."""
    pool = _pool(k_pages, v_pages)
    dev = k_pages.device
    _check((v is None) == (v_pages is None), "v and v_pages must both be given or both be None")
    qs, ks = _tokens(q, "q", k_pages), _tokens(k, "k", k_pages, k_pages.size(2))
    vs = 0 if v is None else _tokens(v, "v", k_pages, k_pages.size(2))
    n = q.size(0)
    _check(k.size(0) == n and (v is None or v.size(0) == n), "q, k and v must have the same number of tokens")
    _check(isinstance(rope, torch.Tensor) and rope.dim() == 2, "rope must have shape [max_position, rope_dim]")
    rope_ptr = _array(rope, "rope", torch.float32, tuple(rope.shape), dev)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _check(isinstance(q_out, torch.Tensor) and q_out.shape == q.shape, "q_out must have q's shape")
    os_ = _tokens(q_out, "q_out", k_pages)
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        _check(w is None or (isinstance(w, torch.Tensor) and w.dim() == 1 and w.dtype == k_pages.dtype
                             and w.device == dev and w.is_contiguous() and w.numel() > 0),
               f"{name} must be a contiguous 1-D tensor of the pages' dtype and device")
        weights += [None, 0] if w is None else [w.data_ptr(), w.numel()]
    g = _geometry(k_pages, rope.size(1), v is None)
    with torch.cuda.device(dev):
        rc = N.lib().ztcp_append_tokens(
            q.data_ptr(), qs, q_out.data_ptr(), os_, k.data_ptr(), ks, None if v is None else v.data_ptr(), vs, n,
            q.size(1), C.byref(pool), C.byref(g), _array(slots, "slots", torch.int64, (n,), dev),
            _array(positions, "positions", torch.int32, (n,), dev), rope_ptr, rope.size(0), *weights, eps,
            int(interleaved), _stream(dev))
    _raise(rc, "append_tokens")
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, q_starts: torch.Tensor, *, scale: float | None = None,
                    max_q_len: int | None = None, return_lse: bool = False, out: torch.Tensor | None = None):
    """Softmax attention of the new tokens ``q`` [rows, q_heads, d] over their
    sequences' pages: the i-th of a sequence's n new tokens sees its tokens up
    to ``kv_len - n + i``, query head h reads KV head ``h // (q_heads //
    kv_heads)``.  Returns ``out`` [rows, q_heads, d] (allocated unless given)
    and, with ``return_lse``, the float32 log-sum-exp [rows, q_heads].

    ``scale`` defaults to ``d ** -0.5``.  ``max_q_len`` is a bound on a
    sequence's new tokens if the caller knows one; 1 spares a decoding step
    the prompt kernel's launch.  A row that sees no token gets zeros and
    -inf; rows of no sequence keep what ``out`` holds (in an ``out`` and an
    lse allocated here, anything)."""
    _check(v_pages is not None, "paged_attention needs K and V pages (single-buffer pages have none)")
    pool = _pool(k_pages, v_pages)
    dev = k_pages.device
    qs = _tokens(q, "q", k_pages)
    n, heads = q.size(0), q.size(1)
    batch = _batch(page_table, kv_lens, q_starts, n, max_q_len, dev)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    out_ptr = _array(out, "out", q.dtype, tuple(q.shape), dev)
    lse = torch.empty((n, heads), dtype=torch.float32, device=dev) if return_lse else None
    g = _geometry(k_pages, 0, False)
    with torch.cuda.device(dev):
        need = N.lib().ztcp_paged_attention_workspace(C.byref(batch), C.byref(pool), C.byref(g), heads)
        if need == C.c_size_t(-1).value:
            _raise(N.EINVAL if N.last_error() else N.EHIP, "paged_attention")
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        rc = N.lib().ztcp_paged_attention(q.data_ptr(), qs, out_ptr, lse.data_ptr() if return_lse else None, heads,
                                          C.byref(pool), C.byref(batch), C.byref(g),
                                          k_pages.size(3) ** -0.5 if scale is None else scale,
                                          work.data_ptr() if need else None, need, _stream(dev))
    _raise(rc, "paged_attention")
    return (out, lse) if return_lse else out


def attention_mass(q: torch.Tensor, lse: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor,
                   kv_lens: torch.Tensor, q_starts: torch.Tensor, mass: torch.Tensor, *, scale: float | None = None,
                   decay: float = 1.0, max_q_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``decay * mass`` plus the attention weight that the pages received from
    the new tokens: [sequences, kv_heads, pages of the table] float32, the sum
    of ``exp(scale * q . k - lse)`` over a KV head's query rows and the page's
    tokens that they see.  ``q``, ``lse`` and ``scale`` as in
    ``paged_attention``.  ``out`` may be ``mass`` itself."""
    pool = _pool(k_pages, None)
    dev = k_pages.device
    qs = _tokens(q, "q", k_pages)
    n, heads = q.size(0), q.size(1)
    batch = _batch(page_table, kv_lens, q_starts, n, max_q_len, dev)
    shape = (page_table.size(0), k_pages.size(2), page_table.size(1))
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    g = _geometry(k_pages, 0, False)
    with torch.cuda.device(dev):
        rc = N.lib().ztcp_attention_mass(q.data_ptr(), qs, _array(lse, "lse", torch.float32, (n, heads), dev), heads,
                                         C.byref(pool), C.byref(batch), C.byref(g),
                                         k_pages.size(3) ** -0.5 if scale is None else scale,
                                         _array(mass, "mass", torch.float32, shape, dev), decay,
                                         _array(out, "out", torch.float32, shape, dev), _stream(dev))
    _raise(rc, "attention_mass")
    return out


class Eviction(NamedTuple):
    """What ``evict_pages`` leaves of the sequences and what it takes."""

    page_table: torch.Tensor   # [sequences, pages] int32: the pages kept, in order, -1 behind them
    mass: torch.Tensor         # [sequences, kv_heads, pages] float32: their accounts, 0 behind them
    kv_lens: torch.Tensor      # [sequences] int32: page_tokens less for each page gone
    evicted: torch.Tensor      # [sequences, pages] int32: the ids given up, in order, -1 behind them
    n_evicted: torch.Tensor    # [sequences] int32


def evict_pages(mass: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor, *, page_tokens: int, budget: int,
                sink: int = 1, recent: int = 1, in_place: bool = False) -> Eviction:
    """The pages that each sequence gives up: all but its first ``sink`` and
    last ``recent`` may go, and those with the least ``mass`` (summed over the
    heads in 64 bits; of equal ones the first) go until ``budget`` pages are
    left or none may go.  ``in_place`` updates ``mass``, ``page_table`` and
    ``kv_lens`` themselves.

    ``descriptors[result.evicted[s, :n]]`` are then the descriptors of those
    pages (``pages.build_descriptors`` of the whole pool) for ``pages.egress``."""
    dev = mass.device if isinstance(mass, torch.Tensor) else None
    _check(dev is not None and mass.is_cuda and mass.dim() == 3,
           "mass must be a HIP tensor [sequences, kv_heads, pages]")
    stride = _table(page_table, "page_table", dev)
    s, mp = page_table.shape
    mass_ptr = _array(mass, "mass", torch.float32, (s, mass.size(1), mp), dev)
    lens_ptr = _array(kv_lens, "kv_lens", torch.int32, (s,), dev)
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=dev)  # noqa: E731
    out = Eviction(page_table if in_place else new(s, mp), mass if in_place else torch.empty_like(mass),
                   kv_lens if in_place else new(s), new(s, mp), new(s))
    with torch.cuda.device(dev):
        rc = N.lib().ztcp_evict_pages(mass_ptr, page_table.data_ptr(), stride, lens_ptr, s, mass.size(1), mp,
                                      page_tokens, budget, sink, recent, out.page_table.data_ptr(),
                                      stride if in_place else mp, out.mass.data_ptr(), out.kv_lens.data_ptr(),
                                      out.evicted.data_ptr(), out.n_evicted.data_ptr(), _stream(dev))
    _raise(rc, "evict_pages")
    return out
