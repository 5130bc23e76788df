"""The operators on hot pages in 64 bits, from their formulas, on the CPU.

Each function also returns what the tests' bounds are made of.  A rounding to
a type is off by at most half a step, ``torch.finfo(t).eps / 2`` relative to
the value (fp16 below its smallest normal number: 2^-25 at most).
"""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rotated(x, weight, rope, positions, eps, interleaved):
    """Norm and rotation of [n, heads, d] in 64 bits, and the largest number that a rounding on the way is relative to."""
    x = x.double()
    d, r = x.shape[-1], rope.shape[1]
    if weight is not None:
        w, b = weight.double(), d - weight.numel()
        t = x[..., b:]
        x = torch.cat([x[..., :b], t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * w], -1)
    big = x.abs()
    if r:
        known = (positions >= 0) & (positions < rope.shape[0])
        row = rope.double()[positions.clamp(0, rope.shape[0] - 1).long()]
        row = torch.where(known[:, None], row, math.nan)[:, None]
        c, s = row[..., :r // 2], row[..., r // 2:]
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
        ya, yb = a * c - b * s, b * c + a * s
        m = a.abs() + b.abs()
        if interleaved:
            x = torch.cat([torch.stack([ya, yb], -1).flatten(-2), x[..., r:]], -1)
            big = torch.cat([torch.stack([m, m], -1).flatten(-2), big[..., r:]], -1)
        else:
            x = torch.cat([ya, yb, x[..., r:]], -1)
            big = torch.cat([m, m, big[..., r:]], -1)
    return x, big


def _gather(pages, table_row, length):
    """Tokens of a sequence that are there, and their places in it."""
    t = pages.shape[1]
    at = torch.arange(length)
    ids = table_row[at // t].long()
    there = (ids >= 0) & (ids < pages.shape[0])
    at = at[there]
    return pages[ids[there], at % t].double(), at


def attention(q, k_pages, v_pages, table, lens, starts, scale, weights_of=None):
    """out, lse [rows, heads] in 64 bits and the bounds on their errors; with
    ``weights_of`` = (lse, mass, decay) the accounts and their bound instead."""
    q, k_pages, table, lens, starts = (x.cpu() for x in (q, k_pages, table, lens, starts))
    v_pages = None if v_pages is None else v_pages.cpu()
    rows, heads, d = q.shape
    kv, t = k_pages.shape[2], k_pages.shape[1]
    g, u = heads // kv, HALF[q.dtype]
    cap = table.shape[1] * t
    out, lse = torch.zeros(rows, heads, d, dtype=torch.float64), torch.full((rows, heads), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros(rows, heads, dtype=torch.float64)
    if weights_of:
        given, mass, decay = weights_of[0].cpu().double(), weights_of[1].cpu().double(), weights_of[2]
        acc = mass * decay
        acc_tol = acc.abs() * 2.0 ** -23
    for s in range(lens.numel()):
        r0 = min(max(int(starts[s]), 0), rows)
        n = min(max(int(starts[s + 1]), r0), rows) - r0
        length = min(max(int(lens[s]), 0), cap)
        k, at = _gather(k_pages, table[s], length)
        v = None if v_pages is None else _gather(v_pages, table[s], length)[0]
        if n == 0 or at.numel() == 0:
            continue
        for h in range(heads):
            x = q[r0:r0 + n, h].double()
            kh = k[:, h // g]
            sc = x @ kh.t() * scale
            # a sum of d products in fp32, and its place in the exponent: relative error of a weight
            delta = (d + 8) * 2.0 ** -24 * (x.abs() @ kh.abs().t()).nan_to_num(0, 0, 0).max() * scale + 2.0 ** -20
            seen = at[None] <= length - n + torch.arange(n)[:, None]
            sc = sc.masked_fill(~seen, -math.inf)
            if weights_of:
                z = given[r0:r0 + n, h, None]
                p = torch.where(z == -math.inf, 0.0, torch.exp(sc - torch.where(z == -math.inf, 0.0, z)))
                p = torch.where(seen, p, 0.0)
                rel = delta + z.abs().nan_to_num(0, 0, 0).max() * 2.0 ** -22 + (n * g + t + 8) * 2.0 ** -24
                both = torch.zeros(table.shape[1], dtype=torch.float64).index_add_(0, at // t, p.sum(0))
                acc[s, h // g] += both
                acc_tol[s, h // g] += both * rel
                continue
            z = torch.logsumexp(sc, -1)
            lse[r0:r0 + n, h] = z
            lse_tol[r0:r0 + n, h] = delta + z.abs().nan_to_num(0, 0, 0) * 2.0 ** -21
            p = torch.where(seen, torch.exp(sc - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
            vh = v[:, h // g]
            for i in range(n) if not torch.isfinite(vh).all() else ():   # unseen numbers take no part, whatever they are
                out[r0 + i, h] = (p[i][seen[i], None] * vh[seen[i]]).sum(0)
            clean = vh.nan_to_num(0, 0, 0)
            if torch.isfinite(vh).all():
                out[r0:r0 + n, h] = p @ vh
            size = p @ clean.abs()
            out_tol[r0:r0 + n, h] = (u + 2 * delta) * (1 + u) * size + u * out[r0:r0 + n, h].abs().nan_to_num(0, 0, 0)
            if q.dtype == torch.float16:   # weights below 2^-14 of the largest, and results below it
                out_tol[r0:r0 + n, h] += 2.0 ** -25 * (1 + clean.abs().sum(0))
    if weights_of:
        return acc, acc_tol + acc.abs() * 2.0 ** -23
    return out, lse, out_tol, lse_tol


def evict(mass, table, lens, page_tokens, budget, sink, recent):
    mass, table, lens = mass.cpu(), table.cpu(), lens.cpu()
    s, _, mp = mass.shape
    new_table, evicted = torch.full_like(table, -1), torch.full_like(table, -1)
    new_mass, new_lens, gone = torch.zeros_like(mass), lens.clone(), torch.zeros_like(lens)
    for i in range(s):
        n = min(-(-max(int(lens[i]), 0) // page_tokens), mp)
        score = mass[i].double().sum(0).tolist()
        key = lambda p: (score[p] != score[p], 0.0 if score[p] != score[p] else score[p], p)  # noqa: E731
        may = list(range(min(sink, n), max(n - recent, min(sink, n))))
        out = sorted(sorted(may, key=key)[:max(0, n - budget)])
        kept = [p for p in range(n) if p not in set(out)]
        new_table[i, :len(kept)], evicted[i, :len(out)] = table[i, kept], table[i, out]
        new_mass[i, :, :len(kept)] = mass[i][:, kept]
        new_lens[i] -= len(out) * page_tokens
        gone[i] = len(out)
    return new_table, new_mass, new_lens, evicted, gone
