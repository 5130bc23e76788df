"""Performance cases of the operators on hot KV pages.

A serving step writes the new tokens' keys and values into the hot pages
(append: norms for each head, rotation and the write in one pass), attends
from the new tokens over each sequence's pages (attention), adds the weight
that every page received to its account (mass), and, when a sequence holds
more pages than its budget, gives up the pages with the least weight (evict),
which then go to the cold codec.

Pages are ``[tokens, kv_heads, head_dim]`` of a pool; a page table row lists a
sequence's pages in order, and an entry outside the pool is a page that is not
there (its tokens take no part).  A sequence of length L with n new tokens has
them at its positions L - n .. L - 1; new token i sees positions
j <= L - n + i.  Query head h reads KV head h // group.
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
EPS = 1e-6
MAX_POSITION = 131072


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

def _append(name, n, group, kv_heads, head_dim, rope, page, dtype, *, interleaved=False, single=False, padded=0.0):
    c = dict(op="append", n=n, group=group, kv_heads=kv_heads, head_dim=head_dim, rope=rope, page=page, dtype=dtype,
             interleaved=interleaved, single=single, padded=padded)
    return dict(c, name=name) if name else c


def _attend(name, op, seqs, kv_low, kv_high, q_low, q_high, group, kv_heads, head_dim, page, dtype, *, one_q=0.0,
            missing=0.0, lens=1):
    """``seqs`` sequences, each of ``kv_low..kv_high`` tokens of which
    ``q_low..q_high`` are new (a share of ``one_q`` has one new token);
    ``lens`` seeds the lengths, so that they belong to the case."""
    c = dict(op=op, seqs=seqs, kv_low=kv_low, kv_high=kv_high, q_low=q_low, q_high=q_high, group=group,
             kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, one_q=one_q, missing=missing, lens=lens)
    return dict(c, name=name) if name else c


def _evict(name, seqs, kv_heads, pages_low, pages_high, page, budget, sink, recent, *, lens=1):
    c = dict(op="evict", seqs=seqs, kv_heads=kv_heads, pages_low=pages_low, pages_high=pages_high, page=page,
             budget=budget, sink=sink, recent=recent, lens=lens)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoding step of 32 sequences: a call of a few microseconds, all latency
        _append("append_decode_32", 32, 4, 8, 128, 64, 16, "bf16"),
        # a prompt of 16,384 tokens of the 8-KV-head, 16-token-page geometry: all bandwidth
        _append("append_prompt_16384", 16384, 4, 8, 128, 64, 16, "bf16"),
        # widths that fill no power of two, neighbouring pairs, rows that a padded batch does not keep
        _append("append_odd_1003", 1003, 3, 5, 96, 32, 13, "fp16", interleaved=True, padded=0.05),
        # one sequence decodes one token over a short context: latency
        _attend("attend_one_1500", "attention", 1, 1500, 1500, 1, 1, 4, 8, 128, 16, "bf16"),
        # a decoding batch of mixed contexts up to 16,384 tokens: reading K and V is the work
        _attend("attend_batch_64", "attention", 64, 500, 16384, 1, 1, 4, 8, 128, 16, "bf16"),
        # decoding sequences beside a chunk of a prompt, ragged pages and widths
        _attend("attend_mixed_odd", "attention", 12, 900, 4001, 300, 700, 3, 5, 96, 13, "fp16", one_q=0.8),
        # two long prompts' second chunk of 4,096 tokens over 64-token pages: matrix products are the work
        _attend("attend_chunk_4096", "attention", 2, 8192, 8192, 4096, 4096, 4, 8, 128, 64, "bf16"),
        # the accounts of one decoding step: one sequence, and the mixed batch
        _attend("mass_one_1500", "mass", 1, 1500, 1500, 1, 1, 4, 8, 128, 16, "bf16"),
        _attend("mass_batch_64", "mass", 64, 500, 16384, 1, 1, 4, 8, 128, 16, "bf16"),
        # the accounts that a prompt's chunk leaves behind
        _attend("mass_chunk_2048", "mass", 2, 4096, 4096, 2048, 2048, 4, 8, 128, 16, "bf16"),
        # eight sequences give up a quarter of 256 pages each: latency
        _evict("evict_8x256", 8, 8, 256, 256, 16, 192, 4, 8),
        # a full node's sequences, up to 8,192 pages (131,072 tokens) each
        _evict("evict_128x8192", 128, 8, 1000, 8192, 16, 2048, 4, 32),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "mass", "evict"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "append":
        if rng.random() < 0.2:  # single-buffer pages: one latent vector a token, no V
            return _append(None, _log(rng, 1, 4096), rng.choice([1, 7, 16]), 1, 576, 64, rng.choice([16, 64]), dtype,
                           interleaved=rng.random() < 0.5, single=True)
        d = rng.choice([64, 80, 96, 128, 192, 256])
        kv = rng.randint(1, 8)
        n = min(_log(rng, 1, 16384), (16384 * 48 * 128) // (kv * 6 * d))
        return _append(None, n, rng.randint(1, 8) if kv * d <= 512 else rng.randint(1, 4), kv, d,
                       rng.choice([0, 16, 32, 64]), rng.choice([1, 7, 16, 64]), dtype,
                       interleaved=rng.random() < 0.5, padded=rng.choice([0.0, 0.0, 0.1]))
    if op in ("attention", "mass"):
        d, kv, group = rng.choice([64, 80, 96, 128, 128, 192, 256]), rng.randint(1, 8), rng.choice([1, 2, 3, 4, 6, 8])
        page, lens = rng.choice([1, 7, 13, 16, 16, 32, 64, 100]), rng.randint(1, 1 << 30)
        way = rng.choice(["decode", "decode", "chunk", "mixed"])
        if way == "decode":
            seqs = _log(rng, 1, 96)
            high = _log(rng, 1, min(20000, (260 << 20) // (seqs * kv * d)))
            q = rng.choice([1, 1, 1, 2, 5])
            return _attend(None, op, seqs, rng.randint(0, high), high, min(q, 1), q, group, kv, d, page, dtype,
                           missing=rng.choice([0.0, 0.0, 0.1]), lens=lens)
        high = _log(rng, 16, 8192)
        q = _log(rng, 2, min(4096, high))
        return _attend(None, op, rng.randint(1, 3) if way == "chunk" else rng.randint(2, 8), rng.randint(q, high),
                       high, rng.randint(1, q), q, group if kv * d * group <= 4096 else 1, kv, d, page, dtype,
                       one_q=0.0 if way == "chunk" else 0.7, lens=lens)
    seqs = _log(rng, 1, 128)
    high = _log(rng, 1, 8192)
    return _evict(None, seqs, rng.randint(1, 8), rng.randint(1, high), high, rng.choice([1, 13, 16, 64]),
                  rng.randint(1, high), rng.randint(0, 8), rng.randint(1, 16), lens=rng.randint(1, 1 << 30))


def _lengths(case):
    """[(new tokens, tokens)] of the case's sequences."""
    rng = random.Random(case["lens"])
    out = []
    for i in range(case["seqs"]):
        kv = _log(rng, case["kv_low"], case["kv_high"]) if case["kv_low"] else rng.randint(0, case["kv_high"])
        q = rng.randint(case["q_low"], case["q_high"])
        if rng.random() < case["one_q"] and i:
            q = 1
        out.append((min(q, kv), kv))
    return out


def _page_counts(case):
    rng = random.Random(case["lens"])
    return [_log(rng, case["pages_low"], case["pages_high"]) for _ in range(case["seqs"])]


def work(case):
    if case["op"] == "append":
        kv, d, n = case["kv_heads"], case["head_dim"], case["n"]
        vecs = kv * (case["group"] + (1 if case["single"] else 2))
        return {"bytes": n * (2 * 2 * vecs * d + 4 * case["rope"] + 12), "flops": n * vecs * d * 6}
    if case["op"] == "evict":
        cells = case["seqs"] * max(_page_counts(case))
        return {"bytes": cells * (2 * 4 * case["kv_heads"] + 2 * 4 + 4), "flops": cells * (case["kv_heads"] + 8)}
    kv, d, g, page = case["kv_heads"], case["head_dim"], case["group"], case["page"]
    lens = _lengths(case)
    rows, keys = sum(q for q, _ in lens), sum(t for _, t in lens)
    pairs = g * kv * sum(q * t - q * (q - 1) // 2 for q, t in lens)
    table = 4 * sum(-(-t // page) for _, t in lens)
    if case["op"] == "attention":
        return {"bytes": 2 * 2 * rows * g * kv * d + 4 * rows * g * kv + 2 * 2 * keys * kv * d + table,
                "flops": 4 * d * pairs}
    cells = case["seqs"] * kv * -(-max(max(t for _, t in lens), 1) // page)
    return {"bytes": 2 * rows * g * kv * d + 4 * rows * g * kv + 2 * keys * kv * d + table + 8 * cells,
            "flops": 2 * d * pairs}


# ---- inputs ----------------------------------------------------------------------

def _table(n_positions, rope):
    """cos | sin of each position's angles, from 64 bits."""
    f = 10000.0 ** (-torch.arange(0, rope, 2, dtype=torch.float64, device="cuda") / max(rope, 1))
    a = torch.arange(n_positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    if case["op"] == "append":
        return _prepare_append(case, seed, gen, normal)
    if case["op"] == "evict":
        counts = torch.tensor(_page_counts(case), device="cuda")
        s, mp, page = case["seqs"], int(counts.max()), case["page"]
        # accounts of weight spread over orders of magnitude, and pages that no query has looked at
        mass = torch.exp(3.0 * normal(s, case["kv_heads"], mp))
        mass *= (torch.rand((s, 1, mp), generator=gen, device="cuda") > 0.3)
        inside = torch.arange(mp, device="cuda")[None] < counts[:, None]
        ids = torch.randperm(s * mp, generator=gen, device="cuda").reshape(s, mp)
        ends = torch.randint(1, page + 1, (s,), generator=gen, device="cuda")
        return dict(case=case, mass=(mass * inside[:, None]).contiguous(),
                    table=torch.where(inside, ids, -1).int().contiguous(),
                    lens=((counts - 1) * page + ends).int())
    dt = DTYPES[case["dtype"]]
    lens, page, kv, d, g = _lengths(case), case["page"], case["kv_heads"], case["head_dim"], case["group"]
    s, need = len(lens), [-(-t // page) for _, t in lens]
    mp, n_pages = max(max(need), 1), sum(need) + 5
    cpu = np.random.default_rng(seed)
    ids, table = cpu.permutation(n_pages), np.full((s, mp), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    if case["missing"]:  # pages that are cold at the moment
        table[cpu.random((s, mp)) < case["missing"]] = -1
    rows = sum(q for q, _ in lens)
    state = dict(case=case, q=(1.5 * normal(rows, kv * g, d)).to(dt),
                 k_pages=normal(n_pages, page, kv, d).to(dt),
                 table=torch.from_numpy(table).cuda(),
                 lens=torch.tensor([t for _, t in lens], dtype=torch.int32, device="cuda"),
                 starts=torch.tensor(np.cumsum([0] + [q for q, _ in lens]), dtype=torch.int32, device="cuda"),
                 max_q=max(q for q, _ in lens), scale=d ** -0.5)
    if case["op"] == "attention":
        state["v_pages"] = normal(n_pages, page, kv, d).to(dt)
    else:
        state["mass"] = torch.rand((s, kv, mp), generator=gen, device="cuda") * 4
        state["lse"] = _plain_attention(state, with_output=False)
    return state


def _prepare_append(case, seed, gen, normal):
    dt = DTYPES[case["dtype"]]
    n, g, kv, d, r, page = (case[x] for x in ("n", "group", "kv_heads", "head_dim", "rope", "page"))
    heads = kv * (g + (1 if case["single"] else 2))
    x = normal(n, heads, d).to(dt)  # one projection's output: queries, keys, values side by side
    pages = -(-n // page) + 3
    slots = (torch.randperm(pages, generator=gen, device="cuda")[:, None] * page
             + torch.arange(page, device="cuda")).reshape(-1)[:n].contiguous()
    slots = torch.where(torch.rand(n, generator=gen, device="cuda") < case["padded"], -1, slots)
    start = int(np.random.default_rng(seed).integers(0, MAX_POSITION - n))
    norms = d - r if case["single"] else d
    return dict(case=case, q=x[:, :kv * g], k=x[:, kv * g:kv * (g + 1)],
                v=None if case["single"] else x[:, kv * (g + 1):], slots=slots,
                positions=(start + torch.arange(n, device="cuda")).int(), rope=_table(MAX_POSITION, r),
                q_weight=None if case["single"] else (1 + 0.1 * normal(d)).to(dt),
                k_weight=(1 + 0.1 * normal(norms)).to(dt), k_pages=torch.zeros((pages, page, kv, d), dtype=dt, device="cuda"),
                v_pages=None if case["single"] else torch.zeros((pages, page, kv, d), dtype=dt, device="cuda"))


# ---- one pass --------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "append":
        return _plain_append(state)
    if op == "attention":
        return _plain_attention(state)
    if op == "mass":
        return _plain_mass(state)
    return _plain_evict(state)


def _own(st, op):
    A = _attention_module()
    if op == "append":
        q = A.append_tokens(st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["slots"], st["positions"],
                            st["rope"], q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS,
                            interleaved=st["case"]["interleaved"])
        return [q, st["k_pages"]] + ([] if st["v"] is None else [st["v_pages"]])
    if op == "attention":
        return A.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["starts"],
                                 scale=st["scale"], max_q_len=st["max_q"], return_lse=True)
    if op == "mass":
        return A.attention_mass(st["q"], st["lse"], st["k_pages"], st["table"], st["lens"], st["starts"], st["mass"],
                                scale=st["scale"], max_q_len=st["max_q"])
    c = st["case"]
    return tuple(A.evict_pages(st["mass"], st["table"], st["lens"], page_tokens=c["page"], budget=c["budget"],
                               sink=c["sink"], recent=c["recent"]))


def _normed_rotated(x, weight, st):
    """Norm and rotation of head vectors [n, heads, d], in 32 bits."""
    x, d, r = x.float(), x.shape[-1], st["case"]["rope"]
    if weight is not None:
        b = d - weight.numel()
        tail = x[..., b:]
        tail = tail * torch.rsqrt((tail * tail).mean(-1, keepdim=True) + EPS) * weight.float()
        x = torch.cat([x[..., :b], tail], -1)
    if r == 0:
        return x
    c, s = st["rope"][st["positions"].long()][:, None].split(r // 2, -1)
    if st["case"]["interleaved"]:
        a, b = x[..., :r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_append(st):
    dt, kept = st["q"].dtype, st["slots"] >= 0
    q = _normed_rotated(st["q"], st["q_weight"], st).to(dt)
    k = _normed_rotated(st["k"], st["k_weight"], st).to(dt)
    at = st["slots"][kept]
    st["k_pages"].flatten(0, 1)[at] = k[kept]
    if st["v"] is None:
        return [q, st["k_pages"]]
    st["v_pages"].flatten(0, 1)[at] = st["v"][kept]
    return [q, st["k_pages"], st["v_pages"]]


def _by_sequence(st):
    """Padded scores [s, kv, row, key] in 32 bits (row = new token * group + head in group), what is seen of them, and
    for each [s, new token] its row of q and whether there is one."""
    c, q, starts, lens = st["case"], st["q"], st["starts"].long(), st["lens"].long()
    kv, g, d, page = c["kv_heads"], c["group"], c["head_dim"], c["page"]
    counts, token = starts[1:] - starts[:-1], torch.arange(max(st["max_q"], 1), device="cuda")
    there = token < counts[:, None]
    row = torch.where(there, starts[:-1, None] + token, 0)
    s, n = row.shape
    x = q[row] if q.shape[0] else q.new_zeros((s, n, kv * g, d))
    x = x.float().reshape(s, n, kv, g, d).permute(0, 2, 1, 3, 4).reshape(s, kv, n * g, d)
    k = st["k_pages"][st["table"].long().clamp_min(0)].flatten(1, 2).float()
    key = torch.arange(k.shape[1], device="cuda")
    limit = lens[:, None] - counts[:, None] + token + 1
    limit = torch.where(there, limit, 0)
    seen = (key < limit[..., None]) & (st["table"] >= 0).repeat_interleave(page, 1)[:, None]
    seen = seen[:, :, None].expand(s, n, g, key.numel()).reshape(s, 1, n * g, key.numel())
    scores = torch.matmul(x * st["scale"], k.permute(0, 2, 3, 1).contiguous())
    return scores.masked_fill_(~seen, -math.inf), row, there


def _rows(padded, st, row, there):
    """[s, kv, new token * group, ...] back to the rows of q: [rows, heads, ...]."""
    c = st["case"]
    s, n = row.shape
    x = padded.unflatten(2, (n, c["group"])).transpose(1, 2).flatten(2, 3)
    return x[there]


def _plain_attention(st, with_output=True):
    scores, row, there = _by_sequence(st)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = _rows((top + total.log())[..., 0], st, row, there).contiguous()
    if not with_output:
        return lse
    v = st["v_pages"][st["table"].long().clamp_min(0)].flatten(1, 2).float().transpose(1, 2).contiguous()
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return _rows(o, st, row, there).to(st["q"].dtype).contiguous(), lse


def _plain_mass(st):
    c = st["case"]
    scores, row, there = _by_sequence(st)
    s, n = row.shape
    lse = st["lse"][row] if st["q"].shape[0] else st["lse"].new_zeros((s, n, c["kv_heads"] * c["group"]))
    lse = lse.reshape(s, n, c["kv_heads"], c["group"]).transpose(1, 2).reshape(s, c["kv_heads"], -1, 1)
    lse = torch.where(lse == -math.inf, torch.zeros_like(lse), lse)
    p = scores.sub_(lse).exp_().sum(2)
    return st["mass"] + p.unflatten(2, (-1, c["page"])).sum(-1)


def _plain_evict(st):
    c, mass, table, lens = st["case"], st["mass"], st["table"], st["lens"]
    mp = table.shape[1]
    index = torch.arange(mp, device="cuda")[None]
    n = ((lens + c["page"] - 1) // c["page"]).clamp(0, mp)[:, None]
    may = (index >= c["sink"]) & (index < n - c["recent"])
    score = torch.where(may, mass.double().sum(1), math.inf)
    rank = torch.argsort(torch.argsort(score, dim=1, stable=True), dim=1)
    gone = (may.sum(1, keepdim=True)).minimum((n - c["budget"]).clamp_min(0))
    out = may & (rank < gone)
    kept = ~out & (index < n)
    order = torch.argsort((~kept).int(), dim=1, stable=True)
    left = index < n - gone
    new_table = torch.where(left, table.gather(1, order), -1)
    new_mass = torch.where(left[:, None], mass.gather(2, order[:, None].expand_as(mass)), 0.0)
    order = torch.argsort((~out).int(), dim=1, stable=True)
    evicted = torch.where(index < gone, table.gather(1, order), -1)
    return (new_table, new_mass, (lens - c["page"] * gone[:, 0]).int(), evicted, gone[:, 0].int())


# ---- the definitions in 64 bits --------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, st)
    if case["op"] == "evict":
        return _exact_evict(case, st)
    return _exact_attend(case, st)


def _exact_append(case, st):
    d, r = case["head_dim"], case["rope"]
    # complex numbers turn by multiplication; the angles are those of the 32-bit table that the call is given
    turn = st["rope"][st["positions"].long()].double()
    turn = torch.complex(turn[:, :r // 2], turn[:, r // 2:])[:, None]

    def one(x, weight):
        x = x.double().clone()
        if weight is not None:
            part = x[..., d - weight.numel():]
            part /= (part.square().sum(-1, keepdim=True) / weight.numel() + EPS).sqrt()
            part *= weight.double()
        if r:
            z = x[..., :r]
            pairs = z.unflatten(-1, (r // 2, 2)) if case["interleaved"] else z.unflatten(-1, (2, r // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            x[..., :r] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return x

    out = [one(st["q"], st["q_weight"])]
    for pool, x in ((st["k_pages"], one(st["k"], st["k_weight"])), (st["v_pages"], st["v"])):
        if pool is None:
            continue
        p = pool.double().flatten(0, 1)
        for_ = (st["slots"] >= 0).nonzero()[:, 0]
        p.index_copy_(0, st["slots"][for_], x.double()[for_])
        out.append(p.view(pool.shape))
    return out


def _exact_attend(case, st):
    kv, g, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    if work(case)["flops"] > 2e12:
        return None
    rows = st["q"].shape[0]
    out = torch.zeros((rows, kv * g, d), dtype=torch.float64, device="cuda")
    lse = torch.full((rows, kv * g), -math.inf, dtype=torch.float64, device="cuda")
    mass = st["mass"].double().clone() if case["op"] == "mass" else None
    at = 0
    for i, (n, total) in enumerate(_lengths(case)):
        table = st["table"][i, :-(-total // page)].long()
        where = (table[:, None] * page + torch.arange(page, device="cuda"))
        where = torch.where(table[:, None] < 0, -1, where).reshape(-1)[:total]
        j = (where >= 0).nonzero()[:, 0]
        for h in range(kv if n and j.numel() else 0):
            k = st["k_pages"].flatten(0, 1)[where[j], h].double()
            q = st["q"][at:at + n, h * g:(h + 1) * g].double()
            s = (q.reshape(n * g, d) @ k.t()).reshape(n, g, -1) * case["head_dim"] ** -0.5
            s.masked_fill_((j[None] > total - n + torch.arange(n, device="cuda")[:, None])[:, None], -math.inf)
            if mass is None:
                w = torch.logsumexp(s, -1)
                lse[at:at + n, h * g:(h + 1) * g] = w
                v = st["v_pages"].flatten(0, 1)[where[j], h].double()
                p = torch.nan_to_num(torch.exp(s - w[..., None]))
                out[at:at + n, h * g:(h + 1) * g] = (p.reshape(n * g, -1) @ v).reshape(n, g, d)
            else:
                w = st["lse"][at:at + n, h * g:(h + 1) * g, None].double()
                p = torch.exp(s - torch.where(w == -math.inf, torch.zeros_like(w), w)).sum((0, 1))
                mass[i, h].index_add_(0, j // page, p)
        at += n
    return (out, lse) if mass is None else mass


def _exact_evict(case, st):
    mass, table, lens = (st[x].cpu().numpy() for x in ("mass", "table", "lens"))
    score = mass.astype(np.float64).sum(1)
    new_table, evicted = np.full_like(table, -1), np.full_like(table, -1)
    new_mass, new_lens, gone = np.zeros(mass.shape), lens.copy(), np.zeros_like(lens)
    for i in range(len(lens)):
        n = -(-int(lens[i]) // case["page"])
        may = range(case["sink"], max(n - case["recent"], case["sink"]))
        m = min(len(may), max(0, n - case["budget"]))
        out = sorted(sorted(may, key=lambda p: (score[i, p], p))[:m])
        kept = sorted(set(range(n)) - set(out))
        new_table[i, :len(kept)], evicted[i, :m] = table[i, kept], table[i, out]
        new_mass[i, :, :len(kept)] = mass[i][:, kept]
        new_lens[i], gone[i] = lens[i] - m * case["page"], m
    return tuple(torch.from_numpy(x) for x in (new_table, new_mass, new_lens, evicted, gone))
