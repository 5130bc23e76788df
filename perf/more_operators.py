"""Performance cases of further operators on hot KV pages: page tables, drafted trees and selected pages.

A serving loop whose page tables live on the GPU gives every sequence the pages
that its new tokens need, and the slots and positions that the append takes
(allot); pages of sequences that ended, or of drafts that were not accepted, go
back to the free ones (release).  Drafted tokens that form a tree attend over
their sequence's pages and over their ancestors among themselves (tree).  For
long contexts each page has the bounds of its keys, column by column (bounds);
from them every query picks the pages that may matter most to it (select), and
attends over these alone (selected).

Pages are ``[tokens, kv_heads, head_dim]`` of a pool; a page table row lists a
sequence's pages in order, and an entry outside the pool is a page that is not
there (its tokens take no part).  A sequence of length L with n new tokens has
them at its places L - n .. L - 1.  Query head h reads KV head h // group.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _attention_module():
    """The product package's module (the package folder's name is not an identifier)."""
    if "vlx_tee_amd" not in sys.modules:
        root = ROOT / "vlx-tee_amd"
        spec = importlib.util.spec_from_file_location("vlx_tee_amd", root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["vlx_tee_amd"] = mod
        spec.loader.exec_module(mod)
    import vlx_tee_amd.attention as attention

    return attention


# ---- cases -----------------------------------------------------------------------

def _allot(name, seqs, kv_low, kv_high, q_low, q_high, page, *, one_q=0.0, free=1.0, room=1.0, counted=False, lens=1):
    """``seqs`` sequences of ``kv_low..kv_high`` tokens get ``q_low..q_high`` more (a share of ``one_q`` gets one); of the
    pages that they need the share ``free`` is there, of the rows the share ``room``; ``counted``: positions go on from the
    sequences' own counts."""
    c = dict(op="allot", seqs=seqs, kv_low=kv_low, kv_high=kv_high, q_low=q_low, q_high=q_high, page=page, one_q=one_q,
             free=free, room=room, counted=counted, lens=lens)
    return dict(c, name=name) if name else c


def _release(name, seqs, kv_low, kv_high, spare, page, *, ended=0.0, lens=1):
    """Sequences of ``kv_low..kv_high`` tokens hold up to ``spare`` pages more than they need; a share of ``ended`` has
    ended and needs none."""
    c = dict(op="release", seqs=seqs, kv_low=kv_low, kv_high=kv_high, spare=spare, page=page, ended=ended, lens=lens)
    return dict(c, name=name) if name else c


def _attend(name, op, seqs, kv_low, kv_high, q_low, q_high, group, kv_heads, head_dim, page, dtype, *, budget=0, sink=1,
            recent=1, missing=0.0, lens=1):
    """``seqs`` sequences of ``kv_low..kv_high`` tokens of which ``q_low..q_high`` are new."""
    c = dict(op=op, seqs=seqs, kv_low=kv_low, kv_high=kv_high, q_low=q_low, q_high=q_high, group=group, kv_heads=kv_heads,
             head_dim=head_dim, page=page, dtype=dtype, budget=budget, sink=sink, recent=recent, missing=missing, lens=lens)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoding step of 64 sequences, of which every sixteenth or so needs a page: all latency
        _allot("allot_decode_64", 64, 500, 16384, 1, 1, 16),
        # a full node: 2,048 sequences, most of them decoding, the others with prompts of up to 2,048 tokens
        _allot("allot_mixed_2048", 2048, 100, 16384, 64, 2048, 16, one_q=0.75, free=0.9, counted=True),
        # 64 sequences give back the pages of drafts that were not accepted
        _release("release_drafts_64", 64, 500, 8192, 4, 16),
        # a quarter of 512 sequences of up to 65,536 tokens has ended
        _release("release_ended_512", 512, 8192, 65536, 2, 16, ended=0.25),
        # the draft of one sequence over a short context, widths and pages that fill no power of two: latency
        _attend("tree_one_odd_37", "tree", 1, 1501, 1501, 37, 37, 3, 5, 96, 13, "fp16"),
        # drafts of 24 to 64 tokens of 32 sequences of mixed contexts
        _attend("tree_batch_32", "tree", 32, 500, 8192, 24, 64, 4, 8, 128, 16, "bf16"),
        # the bounds of the pages that a decoding step of 64 sequences has written
        _attend("bounds_decode_64", "bounds", 64, 500, 4096, 1, 1, 4, 8, 128, 16, "bf16"),
        # the bounds of a prompt of 65,536 tokens
        _attend("bounds_prompt_65536", "bounds", 1, 65536, 65536, 65536, 65536, 4, 8, 128, 16, "bf16"),
        # a decoding step over long contexts, up to 8,192 pages: reading the bounds is the work
        _attend("select_batch_32", "select", 32, 8192, 131072, 1, 1, 4, 8, 128, 16, "bf16", budget=128, recent=4),
        # every token of a chunk picks its pages, ragged widths
        _attend("select_chunk_odd", "select", 2, 32001, 32001, 2000, 2000, 3, 5, 96, 61, "fp16", budget=32, recent=2),
        # a decoding step over 128 pages of each sequence: reading K and V is the work
        _attend("selected_batch_32", "selected", 32, 4000, 32768, 1, 1, 4, 8, 128, 16, "bf16", budget=128),
        # two prompts' chunks of 1,024 tokens, each of which attends over 16 pages of 64 tokens
        _attend("selected_chunk_1024", "selected", 2, 16384, 16384, 1024, 1024, 4, 8, 128, 64, "bf16", budget=16),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["allot", "release", "tree", "tree", "bounds", "select", "select", "selected", "selected"])
    lens = rng.randint(1, 1 << 30)
    if op == "allot":
        seqs, high, page = _log(rng, 1, 2048), _log(rng, 1, 16384), rng.choice([1, 13, 16, 64])
        q = rng.choice([1, _log(rng, 1, min(4096, 2 ** 20 // seqs))])
        if page == 1:
            high, q = min(high, 4096), min(q, 512)
        low = 1 if seqs < 4 else 0   # not all of them empty or idle
        return _allot(None, seqs, rng.randint(low, high), high, rng.randint(low, q), q, page, one_q=rng.choice([0.0, 0.5]),
                      free=rng.choice([1.0, 0.8, 0.3]), room=rng.choice([1.0, 1.0, 0.7]), counted=rng.random() < 0.5, lens=lens)
    if op == "release":
        seqs, high = _log(rng, 1, 512), _log(rng, 1, 65536)
        page = rng.choice([7, 16, 64])
        return _release(None, seqs, rng.randint(0, high), high, _log(rng, 1, 64), page, ended=rng.choice([0.0, 0.1, 0.5]),
                        lens=lens)
    dtype, page = rng.choice(["bf16", "fp16"]), rng.choice([1, 7, 13, 16, 16, 32, 64, 100])
    d, kv, group = rng.choice([64, 80, 96, 128, 128, 192, 256]), rng.randint(1, 8), rng.choice([1, 2, 3, 4, 6, 8])
    missing = rng.choice([0.0, 0.0, 0.1])
    if op == "tree":
        seqs, nodes = _log(rng, 1, 32), _log(rng, 2, 150)
        most = min(16384, (64 << 20) // (seqs * kv * d), 40_000_000_000 // (4 * d * group * kv * seqs * nodes))
        high = _log(rng, nodes, max(nodes, most))
        return _attend(None, op, seqs, rng.randint(nodes, high), high, rng.randint(1, nodes), nodes, group, kv, d, page, dtype,
                       missing=missing, lens=lens)
    if op == "bounds":
        high = _log(rng, 16, 65536)
        q = rng.choice([1, 1, 5, _log(rng, 1, high)])
        seqs = _log(rng, 1, max(1, min(64, 65536 // high))) if q > 5 else _log(rng, 1, 64)
        high = min(high, max(q, (60 << 20) // (seqs * kv * d)))
        return _attend(None, op, seqs, rng.randint(min(q, high), high), high, rng.randint(1 if seqs < 4 else 0, min(q, high)),
                       min(q, high), group, kv, d, page, dtype, missing=missing, lens=lens)
    sink, recent = rng.randint(0, 3), rng.randint(1, 4)
    budget = max(sink + recent, _log(rng, 4, 200))
    if rng.random() < 0.6:   # decoding
        seqs, q = _log(rng, 1, 32), rng.choice([1, 1, 1, 3])
        low = 1 if seqs < 4 else 0
        if op == "select":
            pages = min(_log(rng, 24, 4096), 131072 // page, (48 << 20) // (seqs * kv * d))
            budget = max(sink + recent, min(budget, pages // 2))   # some choice is left
            return _attend(None, op, seqs, rng.randint((budget + 4) * page, pages * page), pages * page, rng.randint(low, q), q,
                           group, kv, d, page, dtype, budget=budget, sink=sink, recent=recent, missing=missing, lens=lens)
        high = max(q, min(_log(rng, q, 32768), (48 << 20) // (seqs * kv * d)))
        return _attend(None, op, seqs, rng.randint(q, high), high, rng.randint(low, q), q, group, kv, d, page, dtype,
                       budget=max(sink + recent, min(budget, max(1, 2048 // page))), sink=sink, recent=recent, missing=missing,
                       lens=lens)
    page = max(page, 7)
    pages = _log(rng, 24, 512)
    high = pages * page
    q = _log(rng, 2, min(high, 1024))
    budget = max(sink + recent, min(budget, pages // 2, max(1, 1024 // page)))
    if kv * group * d > 4096:
        group = 1
    low = max(q, (budget + 4) * page)
    return _attend(None, op, rng.randint(1, 2), rng.randint(low, high), high, rng.randint(1, q), q, group, kv, d, page, dtype,
                   budget=budget, sink=sink, recent=recent, missing=missing, lens=lens)


def _lengths(case):
    """[(new tokens, tokens)] of the case's sequences; of "allot" the tokens are those before the new ones."""
    rng = random.Random(case["lens"])
    out = []
    for _ in range(case["seqs"]):
        kv = _log(rng, case["kv_low"], case["kv_high"]) if case["kv_low"] else rng.randint(0, case["kv_high"])
        q = rng.randint(case["q_low"], case["q_high"])
        if rng.random() < case.get("one_q", 0.0):
            q = 1
        out.append((q if case["op"] == "allot" else min(q, kv), kv))
    return out


def _holdings(case):
    """[(tokens, pages held)] of the case's sequences."""
    rng = random.Random(case["lens"])
    out = []
    for _ in range(case["seqs"]):
        kv = _log(rng, case["kv_low"], case["kv_high"]) if case["kv_low"] else rng.randint(0, case["kv_high"])
        held = -(-kv // case["page"]) + rng.randint(0, case["spare"])
        out.append((0 if rng.random() < case["ended"] else kv, held))
    return out


def _allotted(case):
    """(pages needed, rows asked for, pages there, rows there, columns of the table)"""
    page, lens = case["page"], _lengths(case)
    need = sum(-(-(t + q) // page) - -(-t // page) for q, t in lens)
    rows = sum(q for q, _ in lens)
    columns = max(1, max(-(-(t + q) // page) for q, t in lens))
    return need, rows, math.ceil(need * case["free"]), max(1, int(rows * case["room"])), columns


def work(case):
    page = case["page"]
    if case["op"] == "allot":
        _, _, pages, rows, _ = _allotted(case)
        s = case["seqs"]
        return {"bytes": rows * 12 + pages * 8 + s * (4 * 6 + (8 if case["counted"] else 0)) + 12, "flops": rows * 4 + s * 8}
    if case["op"] == "release":
        held = _holdings(case)
        cells, gone = case["seqs"] * max(max(h for _, h in held), 1), sum(h - -(-t // page) for t, h in held)
        return {"bytes": 8 * cells + 4 * gone + 8 * len(held) + 8, "flops": cells}
    kv, d, g = case["kv_heads"], case["head_dim"], case["group"]
    lens = _lengths(case)
    rows, keys = sum(q for q, _ in lens), sum(t for _, t in lens)
    table = 4 * sum(-(-t // page) for _, t in lens)
    if case["op"] == "bounds":
        touched = [(t - max(t - q, 0) // page * page if q else 0) for q, t in lens]
        pages = sum(-(-x // page) for x in touched)
        return {"bytes": 2 * kv * d * (sum(touched) + 2 * pages) + 4 * pages, "flops": 2 * kv * d * sum(touched)}
    if case["op"] == "tree":
        return {"bytes": 4 * rows * g * kv * d + 4 * rows * g * kv + 4 * keys * kv * d + table + 8 * rows,
                "flops": 4 * d * g * kv * sum(q * (t - q) + q * (q + 1) // 2 for q, t in lens)}
    pages = sum(-(-t // page) for q, t in lens if q)
    seen = [-(-(t - q + i + 1) // page) for q, t in lens for i in range(q)]
    picked = sum(min(x, case["budget"]) for x in seen)
    if case["op"] == "select":
        return {"bytes": 2 * rows * g * kv * d + 4 * pages * kv * d + 4 * pages + 4 * rows * kv * case["budget"],
                "flops": 4 * d * g * kv * sum(seen)}
    read, at = 0, 0
    for q, t in lens:
        read += min(t, page * sum(min(x, case["budget"]) for x in seen[at:at + q]))
        at += q
    return {"bytes": 4 * rows * g * kv * d + 4 * rows * g * kv + 4 * read * kv * d + 4 * rows * kv * case["budget"],
            "flops": 4 * d * g * kv * picked * page}


# ---- inputs ----------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    cpu = np.random.default_rng(seed)
    if case["op"] == "allot":
        return _prepare_allot(case, cpu)
    if case["op"] == "release":
        return _prepare_release(case, cpu)
    dt = DTYPES[case["dtype"]]
    lens, page, kv, d, g = _lengths(case), case["page"], case["kv_heads"], case["head_dim"], case["group"]
    s, need = len(lens), [-(-t // page) for _, t in lens]
    mp, n_pages = max(max(need), 1), sum(need) + 5
    ids, table = cpu.permutation(n_pages), np.full((s, mp), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    if case["missing"]:  # pages that are cold at the moment
        table[cpu.random((s, mp)) < case["missing"]] = -1
    rows = sum(q for q, _ in lens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    state = dict(case=case, table=torch.from_numpy(table).cuda(), lens=i32([t for _, t in lens]),
                 starts=i32(np.cumsum([0] + [q for q, _ in lens])), max_q=max(q for q, _ in lens), scale=d ** -0.5)
    if case["op"] == "bounds":
        state["k_pages"] = normal(n_pages, page, kv, d).to(dt)
        state["bounds"] = torch.zeros((n_pages, 2, kv, d), dtype=dt, device="cuda")
        return state
    state["q"] = (1.5 * normal(rows, kv * g, d)).to(dt)
    if case["op"] == "select":   # a page's keys lie around a point of their own
        middle, width = normal(n_pages, 1, kv, d), 0.7 + normal(n_pages, 1, kv, d).abs()
        state["bounds"] = torch.cat([middle - width, middle + width], 1).to(dt).contiguous()
        return state
    state["k_pages"], state["v_pages"] = normal(n_pages, page, kv, d).to(dt), normal(n_pages, page, kv, d).to(dt)
    if case["op"] == "tree":
        words = max(1, -(-state["max_q"] // 64))
        state["tree"] = torch.from_numpy(_trees([q for q, _ in lens], words, cpu)).cuda()
        return state
    # the first and the last pages that a row sees, and others at random
    limit = (state["lens"] - state["starts"].diff()).long()
    seq = torch.repeat_interleave(torch.arange(s, device="cuda"), state["starts"].diff().long())
    last = (limit[seq] + torch.arange(rows, device="cuda") - state["starts"].long()[seq]) // page
    k = case["budget"]
    chance = torch.rand((rows, kv, mp), generator=gen, device="cuda")
    column = torch.arange(mp, device="cuda")
    chance.masked_fill_((column < case["sink"])[None, None], 2.0)
    chance.masked_fill_((column > last[:, None] - case["recent"])[:, None], 2.0)
    chance.masked_fill_((column > last[:, None])[:, None], -1.0)
    best, at = chance.topk(min(k, mp), dim=-1)
    at = torch.where(best < 0, mp, at).sort(-1).values
    at = torch.nn.functional.pad(torch.where(at == mp, -1, at), (0, max(0, k - mp)), value=-1)
    state["selected"] = at.int().contiguous()
    return state


def _prepare_allot(case, cpu):
    page, lens = case["page"], _lengths(case)
    need, _, pages, rows, mp = _allotted(case)
    held = [-(-t // page) for _, t in lens]
    ids, table, at = cpu.permutation(sum(held) + need), np.full((len(lens), mp), -1, np.int32), 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    free = np.full(sum(held) + need, -1, np.int32)   # room for every page of the pool
    free[:pages] = ids[at:at + pages]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    evicted = cpu.integers(0, 3, len(lens)) * page
    return dict(case=case, table=torch.from_numpy(table).cuda(), lens=i32([t for _, t in lens]),
                wanted=i32([q for q, _ in lens]), free=torch.from_numpy(free).cuda(), n_free=i32([pages]), rows=rows,
                counts=i32([t + e for (_, t), e in zip(lens, evicted)]) if case["counted"] else None)


def _prepare_release(case, cpu):
    held = _holdings(case)
    mp, total = max(max(h for _, h in held), 1), sum(h for _, h in held)
    ids, table, at = cpu.permutation(total + 100), np.full((len(held), mp), -1, np.int32), 0
    for i, (_, n) in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    free = np.full(total + 100, -1, np.int32)
    free[:100] = ids[at:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(case=case, table=torch.from_numpy(table).cuda(), lens=i32([t for t, _ in held]),
                free=torch.from_numpy(free).cuda(), n_free=i32([100]))


def _trees(counts, words, cpu):
    """A random tree for each sequence: what a token sees of its own draft is its line of ancestors and itself."""
    out, at = np.zeros((sum(counts), words), np.uint64), 0
    for n in counts:
        for i in range(n):
            parent = int(cpu.integers(max(-1, i - 9), i))
            if parent >= 0:
                out[at + i] = out[at + parent]
            out[at + i, i // 64] |= np.uint64(1 << (i % 64))
        at += n
    return out.view(np.int64)


# ---- one pass --------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"allot": _plain_allot, "release": _plain_release, "tree": _plain_tree, "bounds": _plain_bounds,
            "select": _plain_select, "selected": _plain_selected}[op](state)


def _own(st, op):
    A, c = _attention_module(), st["case"]
    if op == "allot":
        step = A.allot_pages(st["table"], st["lens"], st["wanted"], st["free"], st["n_free"], page_tokens=c["page"],
                             max_rows=st["rows"], next_positions=st["counts"])
        return [st["table"], *(x for x in step if x is not None)]
    if op == "release":
        return [*A.release_pages(st["table"], st["lens"], st["free"], st["n_free"], page_tokens=c["page"]), st["free"]]
    if op == "bounds":
        return A.page_bounds(st["k_pages"], st["bounds"], st["table"], st["lens"], st["starts"], max_q_len=st["max_q"])
    if op == "tree":
        return A.tree_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["starts"], st["tree"],
                                scale=st["scale"], max_q_len=st["max_q"], return_lse=True)
    if op == "select":
        return A.select_pages(st["q"], st["bounds"], st["table"], st["lens"], st["starts"], page_tokens=c["page"],
                              budget=c["budget"], sink=c["sink"], recent=c["recent"], max_q_len=st["max_q"])
    return A.selected_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["starts"], st["selected"],
                                scale=st["scale"], return_lse=True)


def _plain_allot(st):
    page, table, free = st["case"]["page"], st["table"], st["free"]
    mp, dev = table.shape[1], table.device
    lens = st["lens"].long().clamp(0, mp * page)
    want = st["wanted"].long().clamp_min(0)
    want = torch.where(lens + want <= mp * page, want, 0)   # no more than the table's columns hold
    have = (lens + page - 1) // page
    need = (lens + want + page - 1) // page - have
    rows_upto, pages_upto = want.cumsum(0), need.cumsum(0)
    there = st["n_free"].long()
    served = (rows_upto <= st["rows"]) & ((need == 0) | (pages_upto <= there))
    granted, taken = torch.where(served, want, 0), torch.where(served, need, 0)
    column = torch.arange(mp, device=dev)
    nth = column - have[:, None]   # of the sequence's new pages; the free ones are taken from the end
    fresh = (nth >= 0) & (nth < taken[:, None])
    at = there - 1 - (pages_upto - need)[:, None] - nth
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    starts = torch.nn.functional.pad(granted.cumsum(0), (1, 0))
    row = torch.arange(st["rows"], device=dev)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp_max(lens.numel() - 1)
    nth = row - starts[seq]
    place = torch.where(row < starts[-1], lens[seq] + nth, 0)
    entry = table[seq, place // page].long()
    slots = torch.where((row < starts[-1]) & (entry >= 0), entry * page + place % page, -1)
    counts = lens if st["counts"] is None else st["counts"].long()
    positions = torch.where(row < starts[-1], counts[seq] + nth, 0)
    out = [table, (lens + granted).int(), (there - taken.sum()).int(), starts.int(), slots, positions.int(), granted.int()]
    return out if st["counts"] is None else [*out, (counts + granted).int()]


def _plain_release(st):
    page, table, free = st["case"]["page"], st["table"], st["free"]
    first = (st["lens"].long().clamp_min(0) + page - 1) // page
    gone = (torch.arange(table.shape[1], device=table.device) >= first[:, None]) & (table >= 0)
    nth = gone.flatten().cumsum(0).reshape(gone.shape) - 1 + st["n_free"].long()
    gone &= nth < free.numel()   # what the list has no room for stays
    free.scatter_(0, nth[gone], table[gone])
    count = gone.sum(1)
    return [torch.where(gone, -1, table), (st["n_free"] + count.sum()).int(), count.int(), free]


def _plain_bounds(st):
    page, table, k = st["case"]["page"], st["table"], st["k_pages"]
    lens, new, mp = st["lens"].long()[:, None], st["starts"].diff().long()[:, None], table.shape[1]
    column = torch.arange(mp, device=table.device)
    written = (new > 0) & (column >= (lens - new) // page) & (column * page < lens) & (table >= 0)
    inside = (lens - column * page)[written]   # tokens that the page has
    ids = table[written].long()
    step = max(1, (1 << 28) // (k.shape[1] * k.shape[2] * k.shape[3]))
    token = torch.arange(page, device=table.device)
    for i in range(0, ids.numel(), step):
        part, behind = k[ids[i:i + step]].float(), (token >= inside[i:i + step, None])[..., None, None]
        st["bounds"][ids[i:i + step], 0] = part.masked_fill(behind, math.inf).amin(1).to(k.dtype)
        st["bounds"][ids[i:i + step], 1] = part.masked_fill(behind, -math.inf).amax(1).to(k.dtype)
    return st["bounds"]


def _plain_tree(st):
    """Padded scores [s, kv, row, key] in 32 bits: row = new token * group + head in group."""
    c, q, starts, lens = st["case"], st["q"], st["starts"].long(), st["lens"].long()
    kv, g, d, page = c["kv_heads"], c["group"], c["head_dim"], c["page"]
    counts, token = starts.diff(), torch.arange(st["max_q"], device="cuda")
    there = token < counts[:, None]
    row = torch.where(there, starts[:-1, None] + token, 0)
    s, n = row.shape
    x = q[row].float().reshape(s, n, kv, g, d).permute(0, 2, 1, 3, 4).reshape(s, kv, n * g, d)
    k = st["k_pages"][st["table"].long().clamp_min(0)].flatten(1, 2).float()
    key = torch.arange(k.shape[1], device="cuda")
    nth = key - (lens - counts)[:, None]   # of the new tokens, below 0: before them
    word = st["tree"][row].gather(2, (nth.clamp(0, 64 * st["tree"].shape[1] - 1) // 64)[:, None].expand(s, n, -1))
    seen = (nth < 0)[:, None] | ((word >> (nth.clamp_min(0) % 64)[:, None] & 1) != 0)
    seen = seen & (key < lens[:, None])[:, None] & (st["table"] >= 0).repeat_interleave(page, 1)[:, None] & there[..., None]
    seen = seen[:, :, None].expand(s, n, g, key.numel()).reshape(s, 1, n * g, key.numel())
    scores = torch.matmul(x * st["scale"], k.permute(0, 2, 3, 1).contiguous()).masked_fill_(~seen, -math.inf)
    o, lse = _softmax(scores, st["v_pages"][st["table"].long().clamp_min(0)].flatten(1, 2).float().transpose(1, 2).contiguous())
    rows = lambda t: t.unflatten(2, (n, g)).transpose(1, 2).flatten(2, 3)[there]  # noqa: E731
    return rows(o).to(q.dtype).contiguous(), rows(lse[..., None])[..., 0].contiguous()


def _softmax(scores, v):
    """softmax(scores) @ v and the log-sum-exp; a row that sees nothing has zeros and -inf.  Overwrites scores."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total), (top + total.log())[..., 0]


def _sequence_of_rows(st):
    """Each row's sequence, and how many of its tokens it sees."""
    starts = st["starts"].long()
    row = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, (st["lens"].long() - starts.diff())[seq] + row - starts[seq] + 1


def _plain_select(st):
    """Scores in 64 bits: pages near the border have to fall on the right side of it."""
    c, q, table = st["case"], st["q"], st["table"]
    kv, g, d, page, k, mp = c["kv_heads"], c["group"], c["head_dim"], c["page"], c["budget"], table.shape[1]
    seq, limit = _sequence_of_rows(st)
    out = torch.full((q.shape[0], kv, k), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(mp, device="cuda")
    for s in range(c["seqs"]):
        rows = (seq == s).nonzero()[:, 0]
        n = rows.numel()
        if n == 0:
            continue
        x = q[rows].double().reshape(n, kv, g, d).transpose(0, 1).reshape(kv, n * g, d)
        b = st["bounds"][table[s].long().clamp_min(0)].double()   # [mp, 2, kv, d]
        low, high = (b[:, i].permute(1, 2, 0).contiguous() for i in range(2))
        score = torch.matmul(x.clamp_min(0), high) + torch.matmul(x.clamp_max(0), low)
        score = score.reshape(kv, n, g, mp).amax(2).transpose(0, 1)
        last = ((limit[rows] - 1) // page)[:, None]
        may = (column <= last) & (table[s] >= 0)
        always = may & ((column < c["sink"]) | (column > last - c["recent"]))
        kind = torch.where(always, 0, torch.where(may, 1, 2))[:, None].expand(n, kv, mp)
        by_score = score.argsort(dim=-1, descending=True, stable=True)
        order = by_score.gather(-1, kind.gather(-1, by_score).argsort(dim=-1, stable=True))[..., :k]
        order = torch.where(kind.gather(-1, order) < 2, order, mp).sort(-1).values
        out[rows, :, :order.shape[-1]] = torch.where(order == mp, -1, order).int()
    return out


def _plain_selected(st):
    c, q, table = st["case"], st["q"], st["table"]
    kv, g, d, page, k = c["kv_heads"], c["group"], c["head_dim"], c["page"], c["budget"]
    seq, limit = _sequence_of_rows(st)
    n = q.shape[0]
    out, lse = torch.empty_like(q), torch.empty((n, kv * g), device="cuda")
    head, token = torch.arange(kv, device="cuda")[None, :, None], torch.arange(page, device="cuda")
    step = max(1, (1 << 28) // (kv * k * page * d))
    for i in range(0, n, step):
        at = st["selected"][i:i + step].long()
        b = at.shape[0]
        entry = table[seq[i:i + step, None, None], at.clamp_min(0)]
        entry = torch.where(at >= 0, entry, -1).long()
        seen = (at[..., None] * page + token < limit[i:i + step, None, None, None]) & (entry >= 0)[..., None]
        keys, values = (pool[entry.clamp_min(0), :, head].float().reshape(b, kv, k * page, d)
                        for pool in (st["k_pages"], st["v_pages"]))
        x = q[i:i + step].float().reshape(b, kv, g, d) * st["scale"]
        scores = torch.matmul(x, keys.transpose(2, 3).contiguous()).masked_fill_(~seen.reshape(b, kv, 1, k * page), -math.inf)
        o, z = _softmax(scores, values)
        out[i:i + step], lse[i:i + step] = o.reshape(b, kv * g, d).to(q.dtype), z.reshape(b, kv * g)
    return out, lse


# ---- the definitions in 64 bits --------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"allot": _exact_allot, "release": _exact_release, "tree": _exact_tree, "bounds": _exact_bounds,
            "select": _exact_select, "selected": _exact_selected}[case["op"]](case, st)


def _exact_allot(case, st):
    page, rows = case["page"], st["rows"]
    table, lens, wanted, free = (st[x].cpu().numpy().astype(np.int64) for x in ("table", "lens", "wanted", "free"))
    counts = lens.copy() if st["counts"] is None else st["counts"].cpu().numpy().astype(np.int64)
    there = int(st["n_free"])
    asked = needed = used = taken = 0
    starts, granted = [0], np.zeros_like(lens)
    slots, positions = np.full(rows, -1, np.int64), np.zeros(rows, np.int64)
    for s in range(len(lens)):
        q = max(int(wanted[s]), 0)
        if lens[s] + q > page * table.shape[1]:
            q = 0
        first, end = -(-int(lens[s]) // page), -(-(int(lens[s]) + q) // page)
        asked += q
        needed += end - first
        if asked <= rows and (end == first or needed <= there):
            for p in range(first, end):
                table[s, p] = free[there - 1 - taken]
                taken += 1
            place = lens[s] + np.arange(q)
            entry = table[s, place // page]
            slots[used:used + q] = np.where(entry >= 0, entry * page + place % page, -1)
            positions[used:used + q] = counts[s] + np.arange(q)
            granted[s] = q
            used += q
        starts.append(used)
    t = lambda x, dt=torch.int32: torch.from_numpy(np.asarray(x, np.int64)).to(dt)  # noqa: E731
    out = [t(table), t(lens + granted), t([there - taken]), t(starts), t(slots, torch.int64), t(positions), t(granted)]
    return out if st["counts"] is None else [*out, t(counts + granted)]


def _exact_release(case, st):
    table, lens, free = (st[x].cpu().numpy() for x in ("table", "lens", "free"))
    table, free, n, count = table.copy(), free.copy(), int(st["n_free"]), np.zeros_like(lens)
    for s in range(len(lens)):
        at = -(-int(lens[s]) // case["page"])
        at = at + np.flatnonzero(table[s, at:] >= 0)[:len(free) - n]
        free[n:n + len(at)] = table[s, at]
        table[s, at] = -1
        count[s] = len(at)
        n += len(at)
    return [torch.from_numpy(table), torch.tensor([n], dtype=torch.int32), torch.from_numpy(count), torch.from_numpy(free)]


def _exact_bounds(case, st):
    page, out = case["page"], st["bounds"].double()
    table, k = st["table"].cpu().numpy(), st["k_pages"]
    for s, (q, t) in enumerate(_lengths(case)):
        for p in range((t - q) // page, -(-t // page)) if q else ():
            if table[s, p] >= 0:
                keys = k[table[s, p], :min(page, t - p * page)].double()
                out[table[s, p], 0], out[table[s, p], 1] = keys.min(0).values, keys.max(0).values
    return out


def _exact_tree(case, st):
    kv, g, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    if work(case)["flops"] > 2e12:
        return None
    tree = st["tree"].cpu().numpy().view(np.uint64)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, total) in enumerate(_lengths(case)):
        bits = np.unpackbits(tree[at:at + n].view(np.uint8).reshape(n, -1), axis=1, bitorder="little")[:, :n].astype(bool)
        sees = torch.cat([torch.ones((n, total - n), dtype=torch.bool), torch.from_numpy(bits)], 1).cuda()
        there = st["table"][i].repeat_interleave(page)[:total] >= 0
        where = (st["table"][i].long() * page).repeat_interleave(page)[:total] + torch.arange(total, device="cuda") % page
        where, sees = where[there], sees[:, there]
        for h in range(kv * g if n and where.numel() else 0):
            k, v = (x.flatten(0, 1)[where, h // g].double() for x in (st["k_pages"], st["v_pages"]))
            z = (st["q"][at:at + n, h].double() @ k.t() * d ** -0.5).masked_fill_(~sees, -math.inf)
            w = torch.logsumexp(z, -1)
            lse[at:at + n, h] = w
            out[at:at + n, h] = torch.where(sees, torch.exp(z - w[:, None]), 0.0) @ v
        at += n
    return out, lse


def _exact_select(case, st):
    """A page's score, sum of max(q low, q high) over the columns, is q . (low + high) / 2 + |q| . (high - low) / 2."""
    kv, g, page, k = case["kv_heads"], case["group"], case["page"], case["budget"]
    table = st["table"].cpu().numpy()
    mp, out, at = table.shape[1], np.full((st["q"].shape[0], kv, k), -1, np.int32), 0
    for s, (n, total) in enumerate(_lengths(case)):
        b = st["bounds"][st["table"][s].long().clamp_min(0)].double()
        middle, half = (b[:, 1] + b[:, 0]) / 2, (b[:, 1] - b[:, 0]) / 2
        last = (total - n + np.arange(n)) // page
        column = np.arange(mp)
        may = (column <= last[:, None]) & (table[s] >= 0)
        always = may & ((column < case["sink"]) | (column > last[:, None] - case["recent"]))
        for h in range(kv if n else 0):
            best = None
            for e in range(g):
                x = st["q"][at:at + n, h * g + e].double()
                z = x @ middle[:, h].t() + x.abs() @ half[:, h].t()
                best = z if best is None else torch.maximum(best, z)
            score = np.where(always, np.inf, np.where(may, best.cpu().numpy(), -np.inf))
            order = np.argsort(-score, axis=1, kind="stable")[:, :k]
            kept = np.sort(np.where(np.take_along_axis(may, order, 1), order, mp), axis=1)
            out[at:at + n, h, :kept.shape[1]] = np.where(kept == mp, -1, kept)
        at += n
    return torch.from_numpy(out)


def _exact_selected(case, st):
    kv, g, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    if work(case)["flops"] > 5e11:
        return None
    rows, k = st["q"].shape[0], case["budget"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at, step = 0, max(1, (1 << 26) // (k * page * d))
    for s, (n, total) in enumerate(_lengths(case)):
        for h in range(kv):
            keys, values = (x[:, :, h].flatten(0, 1) for x in (st["k_pages"], st["v_pages"]))
            for i in range(at, at + n, step):
                end = min(at + n, i + step)
                page_at = st["selected"][i:end, h].long()[..., None]
                ids = st["table"][s].long()[page_at.clamp_min(0)]
                place = page_at * page + torch.arange(page, device="cuda")
                limit = total - n + 1 + torch.arange(i - at, end - at, device="cuda")[:, None, None]
                seen = ((page_at >= 0) & (ids >= 0) & (place < limit)).flatten(1)
                where = (ids.clamp_min(0) * page + torch.arange(page, device="cuda")).flatten(1)
                x = st["q"][i:end, h * g:(h + 1) * g].double() * d ** -0.5
                z = torch.matmul(keys[where].double(), x.transpose(1, 2)).masked_fill_(~seen[..., None], -math.inf)
                w = torch.logsumexp(z, 1)
                lse[i:end, h * g:(h + 1) * g] = w
                p = torch.where(seen[..., None], torch.exp(z - w[:, None]), 0.0)
                out[i:end, h * g:(h + 1) * g] = torch.matmul(p.transpose(1, 2), values[where].double())
        at += n
    return out, lse
