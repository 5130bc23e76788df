"""Attention over a tree of drafted tokens and over selected pages in 64 bits, from the formulas, on the CPU, with the bounds
that the tests hold the kernels to.  A rounding to a type is off by at most half a step, ``HALF`` relative to the value."""
from __future__ import annotations

import math

import torch

from hot_reference import HALF


def softmax_rows(x, k, v, seen, scale, dtype):
    """One head: queries x [n, d] over keys k and values v [t, d] of which row i sees seen[i].  out, lse, and the bounds on
    a kernel's errors.  A score is a sum of d products in fp32, scaled and turned into a power of two: delta bounds the
    relative error of a weight.  Weights are rounded to the pages' type for the product with V (u), their total is not;
    the result is rounded once more.  fp16 weights below 2^-14 of the largest, and results below it, step by 2^-24."""
    n, d = x.shape
    u = HALF[dtype]
    sc = x @ k.t() * scale
    delta = (d + 8) * 2.0 ** -24 * float((x.abs() @ k.abs().t()).nan_to_num(0, 0, 0).max()) * scale + 2.0 ** -20 if k.numel() else 0.0
    sc = sc.masked_fill(~seen, -math.inf)
    z = torch.logsumexp(sc, -1) if k.shape[0] else torch.full((n,), -math.inf, dtype=torch.float64)
    p = torch.where(seen, torch.exp(sc - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
    clean = v.nan_to_num(0, 0, 0)
    if torch.isfinite(v).all():
        out = p @ v
    else:   # what a row does not see takes no part, whatever it is
        out = torch.stack([(p[i][seen[i], None] * v[seen[i]]).sum(0) for i in range(n)])
    tol = (u + 2 * delta) * (1 + u) * (p @ clean.abs()) + u * out.abs().nan_to_num(0, 0, 0)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (1 + clean.abs().sum(0))
    return out, z, tol, delta + z.abs().nan_to_num(0, 0, 0) * 2.0 ** -21


def _rows_of(starts, s, rows):
    r0 = min(max(int(starts[s]), 0), rows)
    return r0, min(max(int(starts[s + 1]), r0), rows) - r0


def _blank(rows, heads, d):
    return (torch.zeros(rows, heads, d, dtype=torch.float64), torch.full((rows, heads), -math.inf, dtype=torch.float64),
            torch.zeros(rows, heads, d, dtype=torch.float64), torch.zeros(rows, heads, dtype=torch.float64))


def tree(q, k_pages, v_pages, table, lens, starts, mask, scale):
    """out, lse [rows, heads] and their bounds; mask [rows, words] int64."""
    q, k_pages, v_pages, table, lens, starts, mask = (x.cpu() for x in (q, k_pages, v_pages, table, lens, starts, mask))
    rows, heads, d = q.shape
    t, kv = k_pages.shape[1:3]
    res = _blank(rows, heads, d)
    for s in range(lens.numel()):
        r0, n = _rows_of(starts, s, rows)
        length = min(max(int(lens[s]), 0), table.shape[1] * t)
        at = torch.arange(length)
        ids = table[s, at // t].long()
        at = at[(ids >= 0) & (ids < k_pages.shape[0])]
        if n == 0 or at.numel() == 0:
            continue
        ids = table[s, at // t].long()
        nth = at - (length - n)                                     # of the new tokens
        bits = torch.tensor([[bool(int(mask[r0 + i, j // 64]) >> (j % 64) & 1) if 0 <= j < 64 * mask.shape[1] else False
                              for j in nth.tolist()] for i in range(n)]).reshape(n, -1) if int(nth.max()) >= 0 else \
            torch.zeros(n, at.numel(), dtype=torch.bool)
        seen = (nth < 0)[None] | bits
        for h in range(heads):
            k, v = (x[ids, at % t, h // (heads // kv)].double() for x in (k_pages, v_pages))
            for full, part in zip(res, softmax_rows(q[r0:r0 + n, h].double(), k, v, seen, scale, q.dtype)):
                full[r0:r0 + n, h] = part
    return res


def bounds(k_pages, out, table, lens, starts, rows=1 << 30):
    """``out`` with the bounds of the pages that hold new tokens."""
    k_pages, out, table, lens, starts = (x.cpu() for x in (k_pages, out.clone(), table, lens, starts))
    t = k_pages.shape[1]
    for s in range(lens.numel()):
        _, n = _rows_of(starts, s, rows)
        length = min(max(int(lens[s]), 0), table.shape[1] * t)
        for p in range(max(length - n, 0) // t, -(-length // t)) if n else ():
            if 0 <= int(table[s, p]) < k_pages.shape[0]:
                keys = k_pages[int(table[s, p]), :min(t, length - p * t)]
                out[int(table[s, p]), 0], out[int(table[s, p]), 1] = keys.amin(0), keys.amax(0)   # NaN if there is one
    return out


def select(q, bounds_, table, lens, starts, page_tokens, budget, sink, recent, out):
    """``out`` with the rows that sequences have."""
    q, b, table, lens, starts, out = (x.cpu() for x in (q, bounds_, table, lens, starts, out.clone()))
    rows, heads, _ = q.shape
    kv = b.shape[2]
    for s in range(lens.numel()):
        r0, n = _rows_of(starts, s, rows)
        length = min(max(int(lens[s]), 0), table.shape[1] * page_tokens)
        ids = table[s].long()
        there = (ids >= 0) & (ids < b.shape[0])
        at = b[torch.where(there, ids, 0)].double()
        for i in range(n):
            limit = length - n + i + 1
            pages = -(-limit // page_tokens) if limit > 0 else 0
            for h in range(kv):
                x = q[r0 + i, h * (heads // kv):(h + 1) * (heads // kv)].double()
                high, low = at[:pages, 1, h], at[:pages, 0, h]
                sign = torch.signbit(x)   # NaN goes to either side and stays NaN
                score = (torch.where(sign, 0.0, x)[:, None] * high + torch.where(sign, x, 0.0)[:, None] * low).sum(-1).amax(0).tolist()
                seen = [p for p in range(pages) if there[p]]
                always = [p for p in seen if p < sink or p >= pages - recent]
                rest = sorted((p for p in seen if p not in always),
                              key=lambda p: (score[p] == score[p], -score[p] if score[p] == score[p] else 0.0, p))
                chosen = sorted(always + rest[:budget - len(always)])
                out[r0 + i, h] = torch.tensor(chosen + [-1] * (budget - len(chosen)), dtype=torch.int32)
    return out


def selected(q, k_pages, v_pages, table, lens, starts, picked, scale):
    """out, lse [rows, heads] and their bounds."""
    q, k_pages, v_pages, table, lens, starts, picked = (x.cpu() for x in (q, k_pages, v_pages, table, lens, starts, picked))
    rows, heads, d = q.shape
    t, kv = k_pages.shape[1:3]
    g = heads // kv
    res = _blank(rows, heads, d)
    for s in range(lens.numel()):
        r0, n = _rows_of(starts, s, rows)
        length = min(max(int(lens[s]), 0), table.shape[1] * t)
        for row in range(r0, r0 + n):
            limit = length - n + row - r0 + 1
            for h in range(kv):
                pages, most = [], -1
                for p in picked[row, h].tolist():
                    if most < p < table.shape[1]:   # an entry that is not above all in front of it lists nothing
                        most = p
                        if 0 <= int(table[s, p]) < k_pages.shape[0]:
                            pages.append(p)
                pages = torch.tensor(pages, dtype=torch.int64)
                place = (pages[:, None] * t + torch.arange(t)).flatten()
                place = place[place < limit]
                if place.numel() == 0:
                    continue
                ids = table[s, place // t].long()
                k, v = (x[ids, place % t, h].double() for x in (k_pages, v_pages))
                seen = torch.ones(g, place.numel(), dtype=torch.bool)
                for full, part in zip(res, softmax_rows(q[row, h * g:(h + 1) * g].double(), k, v, seen, scale, q.dtype)):
                    full[row, h * g:(h + 1) * g] = part
    return res
