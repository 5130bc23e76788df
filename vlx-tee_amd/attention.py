"""Operators on hot KV pages: the steps of a serving engine around the codec.

A step's new tokens enter their pages (``append_tokens``: norms of queries and
keys, position rotation and the write in one pass), attend over their
sequences' pages (``paged_attention``), and add to the account of every page
the attention weight it received (``attention_mass``).  A sequence with more
pages than its budget gives up those with the least weight (``evict_pages``);
their ids select the descriptors that ``pages.egress`` takes to the cold tier,
and pages that ``pages.ingress`` brought back are read like any other.

Where the page tables live on the GPU, ``allot_pages`` gives the new tokens
their pages, slots and positions, and ``release_pages`` takes back what ended or
was drafted in vain; drafts that form a tree attend with ``tree_attention``.
For long contexts ``page_bounds`` keeps bounds of every page's keys,
``select_pages`` finds the pages that may matter most to each query, and
``selected_attention`` attends over these alone.

``append_tokens`` and ``evict_pages`` take single-buffer (latent) pages too;
``paged_attention`` is for pages with K and V, and it and ``attention_mass`` for a
head_dim of at most 256.

Pages are the codec's hot pages: a pool ``[n_pages, page_tokens, kv_heads,
head_dim]`` of float16 or bfloat16, each page contiguous (pages may be padded
or interleaved), RoPE columns leading.  Row ``s`` of ``page_table`` lists
sequence ``s``'s pages in order; an entry outside the pool is a page that is
not there (cold) and takes no part.  ``kv_lens`` counts a sequence's tokens,
the new ones among them, which are rows ``q_starts[s]`` to ``q_starts[s + 1]``
of ``q``.

Every call is enqueued on the current stream of its tensors' device,
synchronizes nothing, and can be recorded into a graph.  No operator has a
gradient (they serve, as the codec does): a tensor that requires one is
refused outside ``torch.no_grad()``, and one that carries a forward-mode
tangent everywhere.  Wrong arguments raise ``ValueError``;
indexes on the device are bounded by the kernels as include/ztcp.h says
(ztcp_append_tokens and the entries after it).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

_binding = None


def _call():
    """The native binding (binding/ztcp_torch.cpp), which checks the arguments, allocates the outputs and calls the library."""
    global _binding
    if _binding is None:
        _binding = N.torch_binding()
    return _binding


def rope_table(max_position: int, rope_dim: int, base: float = 10000.0,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """[max_position, rope_dim] float32: the cosines, then the sines, of each
    position's rope_dim / 2 angles ``position * base ** (-2 i / rope_dim)``.
    The angles are computed in 64 bits: at position 100,000 a 32-bit angle is
    off by up to 2^-8."""
    if max_position <= 0 or rope_dim < 0 or rope_dim % 2:
        raise ValueError("max_position must be positive, rope_dim even")
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
    return _call().append_tokens(q, k, v, k_pages, v_pages, slots, positions, rope, q_weight, k_weight, eps, interleaved,
                                 q_out)


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
    return _call().paged_attention(q, k_pages, v_pages, page_table, kv_lens, q_starts, scale, max_q_len, return_lse, out)


def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   kv_lens: torch.Tensor, q_starts: torch.Tensor, tree_mask: torch.Tensor, *, scale: float | None = None,
                   max_q_len: int | None = None, return_lse: bool = False, out: torch.Tensor | None = None):
    """``paged_attention`` of drafted tokens that form a tree: each of a sequence's n new tokens sees all tokens in
    front of the new ones and, of these, the j-th if bit ``j % 64`` of word ``j // 64`` of its row of ``tree_mask``
    [rows, words] (int64) is set: itself and its ancestors.  Bits from n on are not looked at; new tokens behind the last
    word are not seen; a token whose own bit is not set does not see itself.

    The tokens of a tree are to be appended at the positions of their depths, the length in front of the draft plus the
    number of a token's ancestors, which are not those that ``allot_pages`` lays out."""
    return _call().tree_attention(q, k_pages, v_pages, page_table, kv_lens, q_starts, tree_mask, scale, max_q_len, return_lse,
                                  out)


def page_bounds(k_pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                q_starts: torch.Tensor, *, max_q_len: int | None = None) -> torch.Tensor:
    """Brings ``bounds`` [n_pages, 2, kv_heads, d] (the pages' dtype) up to date for the pages that hold the step's new
    tokens: the least and the greatest number of each column of a page's keys, over all of its tokens; NaN where a key's
    is.  Other pages' bounds are left: for keys that were written otherwise call it with ``q_starts`` that count these as
    new, the accepted tokens of a draft that have been moved, or all tokens of a sequence whose pages ``pages.ingress``
    brought back.  Returns ``bounds``."""
    return _call().page_bounds(k_pages, bounds, page_table, kv_lens, q_starts, max_q_len)


def select_pages(q: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                 q_starts: torch.Tensor, *, page_tokens: int, budget: int, sink: int = 1, recent: int = 1,
                 max_q_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The pages that each new token attends over, for each KV head: [rows, kv_heads, budget] int32 columns of the page
    table, ascending, -1 behind them.  Of the pages that the token sees its first ``sink`` and last ``recent`` are always
    taken, and of the others those with the highest scores: for a query head the most that ``q . k`` can be within the
    page's ``bounds``, the sum of ``max(q, 0) * hi + min(q, 0) * lo``, for a KV head the greatest of its query heads'.
    Scores count in 64 bits, NaN as more than every number; of equal ones the first page is taken.  Pages that are not
    there are not taken.  Rows of no sequence keep what ``out`` holds (in one allocated here, anything).  ``max_q_len`` is
    not made use of."""
    return _call().select_pages(q, bounds, page_table, kv_lens, q_starts, page_tokens, budget, sink, recent, max_q_len, out)


def selected_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                       kv_lens: torch.Tensor, q_starts: torch.Tensor, selected: torch.Tensor, *, scale: float | None = None,
                       max_q_len: int | None = None, return_lse: bool = False, out: torch.Tensor | None = None):
    """``paged_attention`` over a part of the pages: a row's query heads of KV head h see, of the tokens that they would
    see, those of the pages in columns ``selected[row, h]`` ([rows, kv_heads, any number] int32, ascending as
    ``select_pages`` gives them).  Entries outside the table's columns (-1) list nothing, and neither does one that is not
    above all columns in front of it.  The log-sum-exp is over what the row sees here.  ``max_q_len`` is not made use of."""
    return _call().selected_attention(q, k_pages, v_pages, page_table, kv_lens, q_starts, selected, scale, max_q_len,
                                      return_lse, out)


def attention_mass(q: torch.Tensor, lse: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor,
                   kv_lens: torch.Tensor, q_starts: torch.Tensor, mass: torch.Tensor, *, scale: float | None = None,
                   decay: float = 1.0, max_q_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``decay * mass`` plus the attention weight that the pages received from
    the new tokens: [sequences, kv_heads, pages of the table] float32, the sum
    of ``exp(scale * q . k - lse)`` over a KV head's query rows and the page's
    tokens that they see.  ``q``, ``lse`` and ``scale`` as in
    ``paged_attention``.  ``out`` may be ``mass`` itself."""
    return _call().attention_mass(q, lse, k_pages, page_table, kv_lens, q_starts, mass, scale, decay, max_q_len, out)


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

    Of the ids given up, ``gone = result.evicted[s, :n]``, those inside the pool
    select their descriptors (``pages.build_descriptors`` of the whole pool) for
    ``pages.egress``: ``descriptors[gone[gone >= 0].long()]``.  An entry that was
    cold already (a page that is not there) has its account and its turn like
    any other, and is listed as the table had it."""
    return Eviction._make(_call().evict_pages(mass, page_table, kv_lens, page_tokens, budget, sink, recent, in_place))


class Allotment(NamedTuple):
    """What ``allot_pages`` leaves of the sequences and what a step's calls take."""

    kv_lens: torch.Tensor                # [sequences] int32: the new tokens among them
    n_free: torch.Tensor                 # [1] int32: free pages left
    q_starts: torch.Tensor               # [sequences + 1] int32
    slots: torch.Tensor                  # [max_rows] int64: -1 behind the last row
    positions: torch.Tensor              # [max_rows] int32: 0 behind the last row
    granted: torch.Tensor                # [sequences] int32: q_lens, or 0 for a sequence that has to wait
    next_positions: torch.Tensor | None  # [sequences] int32, if they were given


def allot_pages(page_table: torch.Tensor, kv_lens: torch.Tensor, q_lens: torch.Tensor, free_pages: torch.Tensor,
                n_free: torch.Tensor, *, page_tokens: int, max_rows: int, next_positions: torch.Tensor | None = None,
                in_place: bool = False) -> Allotment:
    """Gives every sequence the pages that its ``q_lens`` new tokens need, behind the ``kv_lens`` that it has, and lays
    out the step: where each sequence's rows start, each row's slot and position, as ``append_tokens`` and the
    attention calls take them.

    ``free_pages`` [any number] is a stack of page ids of which the first ``n_free`` [1] are there; pages are taken from
    its end and written into ``page_table``.  A sequence gets all or nothing: it waits (``granted`` 0) if the rows that
    it and the sequences in front ask for exceed ``max_rows``, if it needs a page and the pages that they ask for exceed
    ``n_free``, or if its table row has no column left.  Positions go on from ``next_positions`` (after an eviction a
    sequence's own count is more than its length), from ``kv_lens`` if there are none, one further for each row: a line's,
    not a drafted tree's, whose tokens stand at their depths.  A new token whose page is not there (its last page is cold)
    has slot -1.

    ``page_table`` is written in either case; ``in_place`` updates ``kv_lens``, ``n_free`` and ``next_positions`` too."""
    return Allotment._make(_call().allot_pages(page_table, kv_lens, q_lens, free_pages, n_free, page_tokens, max_rows,
                                               next_positions, in_place))


class Release(NamedTuple):
    """What ``release_pages`` leaves."""

    page_table: torch.Tensor   # [sequences, pages] int32: -1 where a page was given back
    n_free: torch.Tensor       # [1] int32
    n_released: torch.Tensor   # [sequences] int32


def release_pages(page_table: torch.Tensor, kv_lens: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor, *,
                  page_tokens: int, in_place: bool = False) -> Release:
    """Puts the pages that ``kv_lens`` tokens do not reach back onto the stack ``free_pages``, of which the first ``n_free``
    are there: those of a sequence that has ended (``kv_lens`` 0), or of drafted tokens that were not accepted.  Pages go in
    the order of sequences and columns; negative entries are no pages, all others are, and one that occurs twice is given
    back twice; what the stack has no room for stays in the table.  The ids that ``evict_pages`` lists are given back, once
    they have been written out, by ``release_pages(cold.evicted, torch.zeros_like(kv_lens), ...)``.

    ``free_pages`` is written in either case; ``in_place`` updates ``page_table`` and ``n_free`` too."""
    return Release._make(_call().release_pages(page_table, kv_lens, free_pages, n_free, page_tokens, in_place))
