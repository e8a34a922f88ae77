"""Measured cases of the paged KV cache's operators: block tables, slot maps, attention of a batch with a shared prefix.

A serving program that decodes a batch whose sequences start with the same long prompt keeps that prompt's K and V once,
in pages that every sequence's block table names.  Three operators carry it:

  block tables   from the lengths of the requests and the pool's free pages: which page holds which positions of whom
  slot map       from the tables and the lengths of a step: where the K and V row of every new token goes
  attention      every query row over its sequence's keys, the shared prefix read once for the whole batch

Head layouts are those of the shapes the repository is configured for (32 / 8 x 64, 16 / 8 x 128, 16 / 16 x 128).
`own` selects the framework's operators; the plain forms are elementary torch operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
LAYOUTS = {"32/8x64": (32, 8, 64), "16/8x128": (16, 8, 128), "16/16x128": (16, 16, 128)}   # query heads, KV heads, head size


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # admission of a small batch: the smallest call, its time is its launch
        dict(name="tables: 8 requests", op="tables", seqs=8, lo=20, hi=400, prefix=128, page=16, max_pages=32, ragged=1),
        # tables of a large server's whole batch in the smallest pages, some requests longer than others by far
        dict(name="tables: 4096 requests", op="tables", seqs=4096, lo=1, hi=8191, prefix=1024, page=16, max_pages=512, ragged=2),
        # the slot map of a decode step: one new token per sequence
        dict(name="slots: decode 64", op="slots", seqs=64, lo=1, hi=4000, new_lo=1, new_hi=1, tokens=64, page=64,
             max_pages=64, ragged=3),
        # a step that mixes decoding sequences with pieces of prompts; the last rows of the step are padding
        dict(name="slots: mixed 16411", op="slots", seqs=777, lo=0, hi=9000, new_lo=0, new_hi=41, tokens=16411, page=16,
             max_pages=568, ragged=4),
        # two sequences behind a short prefix: the smallest attention call, latency counts
        dict(name="decode: 2 rows", op="attention", heads="32/8x64", seqs=2, prefix=128, lo=1, hi=40, new_lo=1, new_hi=1,
             pad=0, page=16, lse=False, ragged=5),
        # an ordinary decode step: 32 sequences behind a system prompt
        dict(name="decode: 32 rows, prefix 2048", op="attention", heads="32/8x64", seqs=32, prefix=2048, lo=1, hi=512,
             new_lo=1, new_hi=1, pad=0, page=64, lse=False, ragged=6),
        # every query head has its own KV head: nothing is shared inside a row, all of it across the batch
        dict(name="decode: 24 rows, 16 KV heads", op="attention", heads="16/16x128", seqs=24, prefix=3600, lo=1, hi=257,
             new_lo=1, new_hi=1, pad=0, page=16, lse=True, ragged=7),
        # a full batch behind a document, in small pages
        dict(name="decode: 64 rows, prefix 12288", op="attention", heads="16/8x128", seqs=64, prefix=12288, lo=1, hi=1024,
             new_lo=1, new_hi=1, pad=0, page=16, lse=False, ragged=8),
        # the widest decode step behind the longest prefix
        dict(name="decode: 128 rows, prefix 65536", op="attention", heads="32/8x64", seqs=128, prefix=65536, lo=1, hi=2048,
             new_lo=1, new_hi=1, pad=0, page=128, lse=False, ragged=9),
        # verification of drafted tokens: five rows per sequence; the step is padded to 208 rows
        dict(name="verify: 40 x 5 rows", op="attention", heads="16/8x128", seqs=40, prefix=4096, lo=10, hi=600, new_lo=5,
             new_hi=5, pad=8, page=32, lse=True, ragged=10),
        # the requests' own prompts behind a shared document: ragged pieces, causal among themselves
        dict(name="extend: 9 pieces, prefix 8192", op="attention", heads="16/8x128", seqs=9, prefix=8192, lo=1, hi=900,
             new_lo=1, new_hi=900, pad=0, page=64, lse=False, ragged=11),
        # long pieces behind a long document: the largest call, bound by its products
        dict(name="extend: 4 pieces, prefix 32768", op="attention", heads="32/8x64", seqs=4, prefix=32768, lo=500, hi=1100,
             new_lo=500, new_hi=1100, pad=0, page=128, lse=False, ragged=12),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    op = rng.choice(["tables", "slots", "attention", "attention", "attention", "attention"])
    while True:
        page = rng.choice([16, 32, 64, 128, 256])
        seed = rng.randrange(1 << 30)
        if op == "tables":
            hi = _spread(rng, 30, 16000)
            case = dict(op=op, seqs=_spread(rng, 1, 4096), lo=rng.choice([0, 1, max(1, hi // 3)]), hi=hi,
                        prefix=page * rng.choice([0, 0, 1, 5, _spread(rng, 1, 64)]), page=page,
                        max_pages=-(-hi // page) + rng.randrange(0, 9), ragged=seed)
        elif op == "slots":
            hi, new_hi = _spread(rng, 20, 16000), _spread(rng, 1, 300)
            seqs = _spread(rng, 1, 2048)
            new_lo = rng.choice([0, 1, new_hi])
            case = dict(op=op, seqs=seqs, lo=0, hi=hi, new_lo=new_lo, new_hi=new_hi,
                        tokens=seqs * (new_lo + new_hi + 1) // 2 + rng.randrange(0, 40), page=page,
                        max_pages=-(-(hi + new_hi) // page), ragged=seed)
        else:
            form = rng.choice(["decode", "decode", "verify", "extend"])
            new_hi = {"decode": 1, "verify": rng.randrange(2, 9), "extend": _spread(rng, 9, 1100)}[form]
            new_lo = new_hi if form != "extend" else rng.choice([0, 1, new_hi // 2])
            hi = _spread(rng, max(new_hi, 8), 2048)
            case = dict(op=op, heads=rng.choice(sorted(LAYOUTS)),
                        seqs=_spread(rng, 1, {"decode": 128, "verify": 64, "extend": 12}[form]),
                        prefix=page * rng.choice([0, max(1, _spread(rng, 64, 65536) // page), max(1, _spread(rng, 256, 32768) // page)]),
                        lo=max(new_hi, rng.choice([1, hi // 2])), hi=max(hi, new_hi), new_lo=new_lo, new_hi=new_hi,
                        pad=rng.choice([0, 0, rng.randrange(1, 17)]), page=page, lse=rng.random() < 0.4, ragged=seed)
            if sum(_sizes(case)[1]) == 0:
                continue
        w = work(case)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1]:
            return case


def _sizes(case):
    """(tokens in the cache, new tokens) of every request, from the case alone.  For tables the first is the reserved
    length, for slots the cached length before the step, for attention the own length behind the prefix, the step's included."""
    r = random.Random(case["ragged"])
    have = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    new = [r.randint(case.get("new_lo", 0), case.get("new_hi", 0)) for _ in range(case["seqs"])]
    if case["op"] == "attention":
        have = [max(h, n) for h, n in zip(have, new)]
    return have, new


# ------------------------------------------------------------------------------------------------ states
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 1000003 + 17)
    have, new = _sizes(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    shuffled = lambda n: torch.randperm(n, generator=gen, device=DEVICE).to(torch.int32)
    page = case["page"]
    st = dict(case=case, page=page)
    if case["op"] == "tables":
        shift = int(seed) % 7                                    # other inputs for another seed
        have = [max(0, h - shift) for h in have]
        shared = case["prefix"] // page
        need = sum(max(0, -(-h // page) - shared) for h in have)
        pool = shuffled(need + shared + 5)
        st.update(lengths=ints(have), prefix_table=pool[:shared].clone(), free_pages=pool[shared:].clone())
        if own:
            from qimeng_megakernel_b200 import paged
            st["out"] = paged.BlockTables.empty(case["seqs"], case["max_pages"], DEVICE)
        return st
    if case["op"] == "slots":
        room = case["max_pages"]
        tables = shuffled(case["seqs"] * room).view(case["seqs"], room)
        for s, (h, n) in enumerate(zip(have, new)):
            tables[s, -(-(h + n) // page):] = -1
        st.update(tables=tables, kv_lengths=ints(have), new_lengths=ints(new))
        if own:
            from qimeng_megakernel_b200 import paged
            st["out"] = paged.SlotMap.empty(case["seqs"], case["tokens"], DEVICE)
        return st
    heads, kv_heads, size = LAYOUTS[case["heads"]]
    shared = case["prefix"] // page
    pages = [-(-h // page) for h in have]
    room = shared + max(pages) + 1
    pool = shuffled(shared + sum(pages) + 3)
    tables = torch.full((case["seqs"], room), -1, dtype=torch.int32)
    order, at = pool.cpu(), shared
    for s, n in enumerate(pages):
        tables[s, :shared] = order[:shared]
        tables[s, shared:shared + n] = order[at:at + n]
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rows = cu[-1] + case["pad"]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)
    cache = lambda: torch.cat([(normal(min(4096, pool.numel() - i), page, kv_heads, size) * 0.9).to(torch.bfloat16)
                               for i in range(0, pool.numel(), 4096)])
    st.update(q=(normal(rows, heads, size) * 1.5).to(torch.bfloat16), k=cache(), v=cache(), tables=tables.to(DEVICE),
              prefix_table=pool[:shared].clone(), kv_lengths=ints([case["prefix"] + h for h in have]), cu_tokens=ints(cu),
              cu=cu, lengths=[case["prefix"] + h for h in have], prefix=case["prefix"],
              out=torch.zeros(rows, heads, size, dtype=torch.bfloat16, device=DEVICE),
              lse=torch.zeros(rows, heads, dtype=torch.float32, device=DEVICE) if case["lse"] else None)
    if own:
        from qimeng_megakernel_b200 import paged
        st["workspace"] = paged.attention_workspace(st["q"], st["k"], case["seqs"], prefix_len=case["prefix"])
    return st


def run(state):
    case = state["case"]
    if case["op"] == "tables":
        return _tables_own(state) if own else _tables_plain(state)
    if case["op"] == "slots":
        return _slots_own(state) if own else _slots_plain(state)
    return _attention_own(state) if own else _attention_plain(state)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _tables_own(st):
    from qimeng_megakernel_b200 import paged
    got = paged.build_block_tables(st["lengths"], st["free_pages"], page_size=st["page"],
                                   max_pages=st["case"]["max_pages"], prefix_table=st["prefix_table"], out=st["out"])
    return {"tables": got.tables, "used": got.used}


def _slots_own(st):
    from qimeng_megakernel_b200 import paged
    got = paged.build_slot_map(st["tables"], st["kv_lengths"], st["new_lengths"], page_size=st["page"],
                               tokens=st["case"]["tokens"], out=st["out"])
    return {"slots": got.slots, "positions": got.positions, "seq_ids": got.seq_ids, "active": got.active,
            "cu_tokens": got.cu_tokens, "kv_lengths": got.kv_lengths}


def _attention_own(st):
    from qimeng_megakernel_b200 import paged
    out = paged.prefix_attention(st["q"], st["k"], st["v"], st["tables"], st["kv_lengths"], st["cu_tokens"],
                                 prefix_table=st["prefix_table"], prefix_len=st["prefix"], out=st["out"], lse=st["lse"],
                                 workspace=st["workspace"])
    return (out, st["lse"]) if st["lse"] is not None else out


# ------------------------------------------------------------------------------------------------ plain forms
def _tables_plain(st):
    page, room = st["page"], st["case"]["max_pages"]
    shared, free = st["prefix_table"].numel(), st["free_pages"]
    wanted = (st["lengths"].clamp(min=0).long() + page - 1) // page
    n = wanted.clamp(max=room)
    mine = (n - shared).clamp(min=0)
    first = torch.cumsum(mine, 0) - mine
    j = torch.arange(room, device=n.device)
    index = first[:, None] + (j - shared)[None, :]
    got = torch.where(index < free.numel(), free[index.clamp(0, max(0, free.numel() - 1))], torch.full_like(free[:1], -1))
    if shared:
        got = torch.where(j[None, :] < shared, st["prefix_table"][j.clamp(max=shared - 1)][None, :], got)
    tables = torch.where(j[None, :] < n[:, None], got, torch.full_like(free[:1], -1))
    return {"tables": tables.to(torch.int32), "used": torch.stack([mine.sum(), (wanted > room).sum()]).to(torch.int32)}


def _slots_plain(st):
    page, rows = st["page"], st["case"]["tokens"]
    tables, kv = st["tables"], st["kv_lengths"].clamp(min=0).long()
    ends = torch.cumsum(st["new_lengths"].clamp(min=0).long(), 0).clamp(max=rows)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(rows, device=kv.device)
    seq = torch.searchsorted(ends, t, right=True)
    real = t < cu[-1]
    s = seq.clamp(max=kv.numel() - 1)
    pos = kv[s] + t - cu[s]
    entry = tables[s, (pos // page).clamp(max=tables.shape[1] - 1)].long()
    held = real & (pos // page < tables.shape[1]) & (entry >= 0)
    none = torch.full_like(pos, -1)
    return {"slots": torch.where(held, entry * page + pos % page, none),
            "positions": torch.where(real, pos, torch.zeros_like(pos)).to(torch.int32),
            "seq_ids": torch.where(real, s, none).to(torch.int32), "active": held.to(torch.uint8),
            "cu_tokens": cu.to(torch.int32), "kv_lengths": (kv + cu[1:] - cu[:-1]).to(torch.int32)}


def _part(q, k, v, limit, scale):
    """Softmax parts of rows q [H, R, D] over keys k [H, N, D]: (max, sum, weighted values); row r sees keys below limit[r]."""
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    if limit is not None:
        s = s.masked_fill(torch.arange(k.shape[1], device=s.device)[None, None, :] >= limit[None, :, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _attention_plain(st):
    rows, heads, size = st["q"].shape
    page, kv_heads, prefix = st["page"], st["k"].shape[2], st["prefix"]
    group, scale = heads // kv_heads, 1.0 / math.sqrt(size)
    # rows of one KV head: its query heads, token by token
    q = st["q"].float().view(rows, kv_heads, group, size).permute(1, 0, 2, 3).reshape(kv_heads, rows * group, size)
    read = lambda cache, ids, n: cache[ids.long()].reshape(-1, kv_heads, size)[:n].float().transpose(0, 1)
    out = torch.zeros(rows, heads, size, dtype=torch.float32, device=q.device)
    lse = torch.zeros(rows, heads, dtype=torch.float32, device=q.device)
    shared = prefix // page
    if shared:
        kp, vp = read(st["k"], st["prefix_table"], prefix), read(st["v"], st["prefix_table"], prefix)
        step = max(1, (1 << 28) // (kv_heads * prefix))
        parts = [_part(q[:, i:i + step], kp, vp, None, scale) for i in range(0, st["cu"][-1] * group, step)]
        parts = [torch.cat(x, 1) for x in zip(*parts)]
    for s, length in enumerate(st["lengths"]):
        a, b = st["cu"][s], st["cu"][s + 1]
        if a == b:
            continue
        n, mine = b - a, length - prefix
        ids = st["tables"][s, shared:shared + -(-mine // page)]
        limit = mine - n + 1 + torch.arange(n * group, device=q.device) // group
        m, l, o = _part(q[:, a * group:b * group], read(st["k"], ids, mine), read(st["v"], ids, mine), limit, scale)
        if shared:
            m0, l0, o0 = (x[:, a * group:b * group] for x in parts)
            top = torch.maximum(m, m0)
            c, c0 = torch.exp(m - top), torch.exp(m0 - top)
            m, l, o = top, l * c + l0 * c0, o * c + o0 * c0
        back = lambda x: x.view(kv_heads, n, group, -1).permute(1, 0, 2, 3).reshape(n, heads, -1)
        out[a:b] = back(o / l)
        lse[a:b] = back(m + torch.log(l))[..., 0]
    out = out.to(torch.bfloat16)
    return (out, lse) if st["lse"] is not None else out


# ------------------------------------------------------------------------------------------------ 64-bit values
def exact(case, seed):
    """Attention from its definition: every row's whole softmax at once, request by request, in 64 bits.  The tables and
    the slot map are whole numbers, which have no other value than their own."""
    if case["op"] != "attention":
        return None
    st = prepare(case, seed)
    rows, heads, size = st["q"].shape
    page, kv_heads = st["page"], st["k"].shape[2]
    group = heads // kv_heads
    shared = st["prefix"] // page
    out = torch.zeros(rows, heads, size, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(rows, heads, dtype=torch.float64, device=DEVICE)
    for s in range(len(st["lengths"])):
        n = st["cu"][s + 1] - st["cu"][s]
        if n == 0:
            continue
        count = st["lengths"][s]
        ids = torch.cat([st["prefix_table"], st["tables"][s, shared:-(-count // page)]]).long()
        for h in range(kv_heads):
            k = st["k"][ids, :, h].reshape(-1, size)[:count].double()
            v = st["v"][ids, :, h].reshape(-1, size)[:count].double()
            for a in range(0, n, 512):
                b = min(n, a + 512)
                at = slice(st["cu"][s] + a, st["cu"][s] + b)
                mine = slice(h * group, (h + 1) * group)
                scores = torch.einsum("rgd,kd->rgk", st["q"][at, mine].double(), k) / math.sqrt(size)
                place = torch.arange(count, device=DEVICE)
                last = count - n + torch.arange(a, b, device=DEVICE)
                scores.masked_fill_((place[None, :] > last[:, None])[:, None, :], float("-inf"))
                total = torch.logsumexp(scores, dim=-1)
                lse[at, mine] = total
                out[at, mine] = torch.einsum("rgk,kd->rgd", torch.exp(scores - total[..., None]), v)
    return (out, lse) if st["lse"] is not None else out


# ------------------------------------------------------------------------------------------------ work
def work(case):
    have, new = _sizes(case)
    page, seqs = case["page"], case["seqs"]
    if case["op"] == "tables":
        shared = case["prefix"] // page
        mine = sum(max(0, min(-(-h // page), case["max_pages"]) - shared) for h in have)
        return {"bytes": 4 * seqs + 4 * (mine + shared) + 4 * seqs * case["max_pages"] + 8, "flops": 0}
    if case["op"] == "slots":
        touched = sum(((h + n - 1) // page - h // page + 1) if n else 0 for h, n in zip(have, new))
        return {"bytes": 8 * seqs + 4 * touched + 17 * case["tokens"] + 8 * seqs + 4, "flops": 0}
    heads, kv_heads, size = LAYOUTS[case["heads"]]
    rows = sum(new)
    keys = case["prefix"] + sum(h for h, n in zip(have, new) if n)
    seen = sum(n * (case["prefix"] + h - n) + n * (n + 1) // 2 for h, n in zip(have, new))
    return {"bytes": 4 * rows * heads * size + 4 * keys * kv_heads * size + (4 * rows * heads if case["lse"] else 0),
            "flops": 4 * size * heads * seen}
