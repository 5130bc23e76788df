"""Page tables on the GPU from their rules, on the CPU in whole numbers."""
from __future__ import annotations

import torch


def allot(table, lens, wanted, free, n_free, page_tokens, max_rows, counts=None):
    """The table, then the fields of ``Allotment``."""
    table, cols = table.cpu().clone(), table.shape[1]
    lens, wanted, free = lens.cpu().tolist(), wanted.cpu().tolist(), free.cpu().tolist()
    there = min(max(int(n_free), 0), len(free))
    lens = [min(max(x, 0), cols * page_tokens) for x in lens]
    counts = list(lens) if counts is None else counts.cpu().tolist()
    slots, positions, starts, granted = [], [], [0], []
    rows = pages = taken = 0
    for s, (have, q) in enumerate(zip(lens, wanted)):
        q = max(q, 0)
        if have + q > cols * page_tokens:
            q = 0
        first, end = -(-have // page_tokens), -(-(have + q) // page_tokens)
        rows, pages = rows + q, pages + end - first
        if rows > max_rows or (end > first and pages > there):
            q, end = 0, first
        for p in range(first, end):
            taken += 1
            table[s, p] = free[there - taken]
        for i in range(q):
            entry = int(table[s, (have + i) // page_tokens])
            slots.append(entry * page_tokens + (have + i) % page_tokens if entry >= 0 else -1)
            positions.append(counts[s] + i)
        granted.append(q)
        starts.append(starts[-1] + q)
    behind = max_rows - len(slots)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return (table, i32([a + b for a, b in zip(lens, granted)]), i32([there - taken]), i32(starts),
            torch.tensor(slots + [-1] * behind, dtype=torch.int64), i32(positions + [0] * behind), i32(granted),
            i32([a + b for a, b in zip(counts, granted)]))


def release(table, lens, free, n_free, page_tokens):
    """The table, the number of free pages, those released, the stack."""
    table, free, n = table.cpu().clone(), free.cpu().clone(), min(max(int(n_free), 0), free.numel())
    count = torch.zeros(table.shape[0], dtype=torch.int32)
    for s, have in enumerate(lens.cpu().tolist()):
        for p in range(-(-max(have, 0) // page_tokens), table.shape[1]):
            if table[s, p] >= 0 and n < free.numel():
                free[n] = table[s, p]
                table[s, p] = -1
                n += 1
                count[s] += 1
    return table, torch.tensor([n], dtype=torch.int32), count, free
