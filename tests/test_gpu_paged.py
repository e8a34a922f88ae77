"""Paged KV cache on the GPU: block tables and slot maps against plain Python, attention with a shared prefix against its
definition in 64 bits.

Tolerance of the attention, derived per element: the kernel rounds the output once (2^-8 |o|) and every probability once
(2^-8 of it, so 2^-8 A with A = sum_j softmax_j |v_j|); a score is a sum of HD exact products in fp32, scaled once, and its
exponential is good to 2^-14, so a probability is off by at most r = 2 * ((HD + 8) 2^-24 scale max|q||k| + 2^-14) more,
numerator and sum together.  |error| <= 2^-8 |o| + (2^-8 + r)(1 + 2^-6) A.  The logarithm of the sum is off by r + 2^-22 |lse|.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS = {"32/8x64": (32, 8, 64), "16/8x128": (16, 8, 128), "16/16x128": (16, 16, 128), "6/2x64": (6, 2, 64),
         "8/1x128": (8, 1, 128), "16/1x64": (16, 1, 64), "5/1x128": (5, 1, 128), "3/3x64": (3, 3, 64)}


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from qimeng_megakernel_b200 import paged
    return paged


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda:0")


# ------------------------------------------------------------------------------------------------ tables
def plain_tables(lengths, free, page, room, prefix):
    at, rows, cut = 0, [], 0
    for n in lengths:
        want = -(-max(n, 0) // page)
        cut += want > room
        row = []
        for j in range(min(want, room)):
            if j < len(prefix):
                row.append(prefix[j])
            else:
                row.append(free[at] if at < len(free) else -1)
                at += 1
        rows.append(row + [-1] * (room - len(row)))
    return rows, [at, cut]


@pytest.mark.parametrize("seqs,page,shared,room,short", [
    (1, 16, 0, 1, False), (1, 16, 0, 5, False), (3, 64, 2, 7, False), (8, 16, 1, 33, False), (9, 256, 0, 4, True),
    (255, 32, 3, 40, False), (257, 16, 0, 64, True), (2500, 16, 5, 31, False), (5000, 128, 1, 3, False)])
def test_block_tables(paged, seqs, page, shared, room, short):
    r = random.Random(seqs * 31 + page)
    lengths = [r.choice([0, 1, page, page + 1, r.randrange(0, room * page + 1), r.randrange(0, room * page + 3 * page), -4])
               for _ in range(seqs)]
    total = sum(max(0, -(-max(n, 0) // page)) for n in lengths) + 4
    pool = list(range(total + shared))
    r.shuffle(pool)
    prefix, free = pool[:shared], pool[shared:]
    if short:
        free = free[:total // 2]
    rows, used = plain_tables(lengths, free, page, room, prefix)
    got = paged.build_block_tables(ints(lengths), ints(free), page_size=page, max_pages=room,
                                   prefix_table=ints(prefix) if shared else None)
    assert got.used.tolist() == used
    assert got.tables.tolist() == rows


def test_block_tables_with_no_free_page(paged):
    got = paged.build_block_tables(ints([40, 0, 16]), ints([]), page_size=16, max_pages=4, prefix_table=ints([7]))
    assert got.tables.tolist() == [[7, -1, -1, -1], [-1] * 4, [7, -1, -1, -1]]
    assert got.used.tolist() == [2, 0]


def plain_slots(tables, kv, new, page, tokens):
    slots, pos, ids, act, cu, out = [], [], [], [], [0], []
    for s, (have, n) in enumerate(zip(kv, new)):
        have, n = max(have, 0), min(max(n, 0), tokens - cu[-1])
        for i in range(n):
            p = have + i
            entry = tables[s][p // page] if p // page < len(tables[s]) else -1
            slots.append(entry * page + p % page if entry >= 0 else -1)
            pos.append(p); ids.append(s); act.append(int(entry >= 0))
        cu.append(cu[-1] + n); out.append(have + n)
    rest = tokens - cu[-1]
    return dict(slots=slots + [-1] * rest, positions=pos + [0] * rest, seq_ids=ids + [-1] * rest, active=act + [0] * rest,
                cu_tokens=cu, kv_lengths=out)


@pytest.mark.parametrize("seqs,page,most_new,tokens", [
    (1, 16, 1, 1), (1, 16, 3000, 2999), (5, 64, 1, 8), (64, 32, 1, 64), (300, 16, 9, 700), (300, 16, 9, 2000),
    (2047, 128, 2, 2500), (2049, 16, 1, 300), (6000, 256, 3, 7000), (40, 16, 600, 12001)])
def test_slot_map(paged, seqs, page, most_new, tokens):
    r = random.Random(seqs + tokens)
    kv = [r.choice([0, 1, page - 1, page, r.randrange(0, 40 * page), -2]) for _ in range(seqs)]
    new = [r.choice([most_new, 0, r.randrange(0, most_new + 1), -3 if seqs > 5 else most_new]) for _ in range(seqs)]
    room = 30                                          # some positions lie behind the table
    tables = [[r.choice([r.randrange(0, 1 << 20), r.randrange(0, 1 << 20), (1 << 31) - 1, -1]) for _ in range(room)]
              for _ in range(seqs)]
    want = plain_slots(tables, kv, new, page, tokens)
    got = paged.build_slot_map(ints(tables), ints(kv), ints(new), page_size=page, tokens=tokens)
    for name, values in want.items():
        assert getattr(got, name).tolist() == values, name


def test_slot_map_sums_past_32_bits(paged):
    big = (1 << 31) - 1
    got = paged.build_slot_map(ints([[3, 4]] * 4), ints([1, big, 5, 0]), ints([2, big, big, 7]), page_size=16, tokens=5)
    assert got.cu_tokens.tolist() == [0, 2, 5, 5, 5]
    assert got.kv_lengths.tolist() == [3, big, 5, 0]
    assert got.slots.tolist() == [49, 50, -1, -1, -1]
    assert got.positions.tolist() == [1, 2, big, big, big]


# ------------------------------------------------------------------------------------------------ attention
def make_case(heads, page, prefix, own, new, seed=0, pad=0, extra_room=2, q_gap=0):
    """Requests with own[s] tokens behind the prefix, the last new[s] of them rows of the step.  Everything in the pool that no
    request lists, and everything behind a request's last token, is NaN or infinity."""
    H, HK, D = HEADS[heads]
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(seed + 1)
    shared = prefix // page
    pages = [-(-max(n, 0) // page) for n in own]
    total = shared + sum(pages) + 3
    pool = torch.randperm(total, generator=gen, device="cuda:0").to(torch.int32).tolist()
    room = shared + max(pages) + extra_room
    tables, at = [], shared
    bad = float("nan") if seed % 2 else float("inf")
    k = torch.full((total, page, HK, D), bad, dtype=torch.bfloat16, device="cuda:0")
    v = torch.full((total, page, HK, D), bad, dtype=torch.bfloat16, device="cuda:0")
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda:0").to(torch.bfloat16)
    if shared:
        ids = torch.tensor(pool[:shared], device="cuda:0")
        k[ids], v[ids] = normal(shared, page, HK, D), normal(shared, page, HK, D)
    for n, count in zip(own, pages):
        mine = pool[at:at + count]
        at += count
        # entries of the prefix are not read through the table, those behind the last token not at all
        tables.append([1 << 30] * shared + mine + [-7] * (room - shared - count))
        for j, pg in enumerate(mine):
            here = min(page, n - j * page)
            k[pg, :here], v[pg, :here] = normal(here, HK, D), normal(here, HK, D)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    rows = cu[-1] + pad
    q = normal(rows, H + q_gap, D).mul_(1.5)[:, :H]
    return dict(q=q, k=k, v=v, tables=ints(tables), kv=ints([prefix + n for n in own]), cu=ints(cu),
                prefix_table=ints(pool[:shared]) if shared else None, prefix=prefix, page=page,
                own=own, new=new, cu_list=cu, pool=pool)


def call(paged, c, **more):
    return paged.prefix_attention(c["q"], c["k"], c["v"], c["tables"], c["kv"], c["cu"], prefix_table=c["prefix_table"],
                                  prefix_len=c["prefix"], **more)


def definition(c, scale=None):
    """(o, lse, A, r) in 64 bits: the output, the log of the sum, sum softmax |v| and the relative slack of a probability."""
    T, H, D = c["q"].shape
    HK, page = c["k"].shape[2], c["page"]
    scale = 1 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(T, H, D, dtype=torch.float64, device="cuda:0")
    A, lse = torch.zeros_like(o), torch.full((T, H), float("-inf"), dtype=torch.float64, device="cuda:0")
    r = torch.zeros(T, H, 1, dtype=torch.float64, device="cuda:0")
    pool = c["k"].shape[0]
    shared = c["prefix"] // page
    for s, n in enumerate(c["new"]):
        count = c["prefix"] + c["own"][s]
        if n == 0 or count <= 0:
            continue
        ids = (c["prefix_table"].tolist() if shared else []) + c["tables"][s].tolist()[shared:]
        ids = ids[:-(-count // page)]
        held = torch.tensor([0 <= i < pool for i in ids], device="cuda:0")
        at = torch.tensor([i if 0 <= i < pool else 0 for i in ids], dtype=torch.int64, device="cuda:0")
        get = lambda x: torch.where(held[:, None, None, None], x[at], torch.zeros_like(x[:1])).reshape(-1, HK, D)[:count].double()
        k, v = get(c["k"]), get(c["v"])
        for i in range(n):
            lim = count - n + i + 1
            if lim <= 0:
                continue
            t = c["cu_list"][s] + i
            q = c["q"][t].double().view(HK, H // HK, D)
            x = torch.einsum("hgd,khd->hgk", q, k[:lim]) * scale
            p = torch.softmax(x, -1)
            o[t] = torch.einsum("hgk,khd->hgd", p, v[:lim]).reshape(H, D)
            A[t] = torch.einsum("hgk,khd->hgd", p, v[:lim].abs()).reshape(H, D)
            lse[t] = torch.logsumexp(x, -1).reshape(H)
            top = torch.einsum("hgd,khd->hgk", q.abs(), k[:lim].abs())
            top = torch.where(torch.isfinite(top), top, 0).amax(-1).reshape(H, 1) * scale
            r[t] = 2 * ((D + 8) * 2.0 ** -24 * top + 2.0 ** -14)
    return o, lse, A, r


def compare(c, out, lse=None, scale=None):
    o, want_lse, A, r = definition(c, scale)
    real = c["cu_list"][-1]
    err = (out.double() - o).abs()[:real]
    tol = (2.0 ** -8 * o.abs() + (2.0 ** -8 + r) * (1 + 2.0 ** -6) * A)[:real]
    worst = (err - tol).max().item() if real else 0.0
    assert not torch.isnan(out[:real].float()).any()
    assert worst <= 0.0, f"outside the derived tolerance by {worst:.3g} (largest error {err.max().item():.3g})"
    if lse is not None and real:
        none = torch.isinf(want_lse[:real])
        assert torch.equal(torch.isinf(lse[:real]), none)
        gap = (lse.double() - want_lse).abs()[:real][~none]
        slack = (r[..., 0] + 2.0 ** -22 * want_lse.abs())[:real][~none]
        assert (gap <= slack).all(), f"lse off by {gap.max().item():.3g}"


SHAPES = [  # prefix, own lengths, new rows
    (0, [1], [1]), (0, [17], [1]), (0, [300, 1, 64, 65], [1, 1, 1, 1]), (256, [1], [1]), (256, [5, 130], [1, 1]),
    (512, [33] * 9, [1] * 9), (256, [40, 3, 200, 7], [5, 3, 0, 7]), (0, [40, 128, 129], [40, 128, 129]),
    (768, [90, 200, 1, 31], [70, 131, 1, 2]), (256, [0, 3], [0, 1]), (1280, [257], [257]), (2304, [20] * 33, [1] * 33)]


@pytest.mark.parametrize("heads", sorted(HEADS))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_against_definition(paged, heads, shape):
    prefix, own, new = SHAPES[shape]
    page = [16, 64, 256, 32, 128, 16][(shape + sorted(HEADS).index(heads)) % 6]
    c = make_case(heads, page, prefix, own, new, seed=shape, pad=shape % 3)
    H = c["q"].shape[1]
    lse = torch.full((c["q"].shape[0], H), 7.0, device="cuda:0")
    out = torch.full_like(c["q"], 3.0)
    got = call(paged, c, out=out, lse=lse)
    assert got is out
    compare(c, out, lse)
    real = c["cu_list"][-1]
    assert (out[real:] == 3.0).all() and (lse[real:] == 7.0).all(), "rows behind the last request were written"


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128"])
def test_attention_page_sizes_and_edges(paged, heads, page):
    for own in ([page - 1], [page], [page + 1], [2 * page + 3, page, 1]):
        compare(c := make_case(heads, page, page, own, [1] * len(own), seed=page + len(own)), call(paged, c))
    compare(c := make_case(heads, page, 2 * page, [page + 9, 5], [page + 3, 5], seed=3), call(paged, c))


def test_rows_that_see_nothing_or_part_of_the_prefix(paged):
    """More rows than tokens in the cache: the first rows see nothing; lengths inside the prefix: those see part of it."""
    for heads in ("32/8x64", "16/8x128"):
        H, HK, D = HEADS[heads]
        c = make_case(heads, 32, 64, [40, 10, 3], [6, 1, 40], seed=2)
        c["own"] = [-61, 10, -30]                                  # 3 and 34 tokens in the cache, 64 of them would be shared
        c["kv"] = ints([64 + n for n in c["own"]])
        lse = torch.empty(47, H, device="cuda:0")
        out = call(paged, c, lse=lse)
        compare(c, out, lse)
        assert (out[:3] == 0).all() and torch.isinf(lse[:3]).all() and (out[3:7] != 0).any()
        c["own"] = [-64 - 9, 10, -64]                              # a length of zero and one below it
        c["kv"] = ints([64 + n for n in c["own"]])
        out = call(paged, c, lse=lse)
        compare(c, out, lse)
        assert (out[:6] == 0).all() and (out[7:] == 0).all()


def test_pages_outside_the_pool_read_as_zeros(paged):
    for heads in ("32/8x64", "16/16x128"):
        c = make_case(heads, 16, 64, [70, 33], [1, 20], seed=4)
        t = c["tables"].tolist()
        t[0][5], t[1][4] = -1, c["k"].shape[0]
        c["tables"] = ints(t)
        p = c["prefix_table"].tolist()
        p[1] = 1 << 29
        c["prefix_table"] = ints(p)
        compare(c, call(paged, c))
        # lengths behind the table: what it holds is seen, no more
        c = make_case(heads, 16, 0, [32, 48], [1, 3], seed=4, extra_room=0)
        c["kv"] = ints([1 << 30, 48])
        want = call(paged, dict(c, kv=ints([48, 48]), tables=ints([c["tables"].tolist()[0][:2] + [-7], c["tables"].tolist()[1]])))
        assert torch.equal(call(paged, c), want)


def test_strided_rows_scale_and_extreme_scores(paged):
    c = make_case("16/8x128", 32, 128, [50, 3], [1, 2], seed=6, q_gap=4)
    assert not c["q"].is_contiguous()
    wide = torch.full((3, 20, 128), 9.0, dtype=torch.bfloat16, device="cuda:0")
    out = call(paged, c, out=wide[:, :16], scale=0.3)
    compare(c, out, scale=0.3)
    assert (wide[:, 16:] == 9.0).all()
    # scores of several hundred: the maximum carries, nothing overflows
    c = make_case("32/8x64", 64, 640, [90, 20, 7], [1, 1, 7], seed=7)
    c["q"] = c["q"] * 40
    compare(c, call(paged, c))


def test_scores_of_minus_infinity_and_rising_maxima(paged):
    """Keys that make a score minus infinity count as absent; keys that grow along the sequence move the maximum in every block."""
    c = make_case("32/8x64", 16, 256, [300, 40], [1, 30], seed=8)
    c["q"] = c["q"].abs()
    ramp = torch.linspace(0.01, 6, c["k"].shape[0], device="cuda:0").to(torch.bfloat16)
    order = torch.tensor(c["pool"], device="cuda:0")
    c["k"][order] = c["k"][order].abs() * ramp[:, None, None, None]
    compare(c, call(paged, c))
    c["k"][c["pool"][1]] = float("-inf")                           # a page of the prefix
    compare(c, call(paged, c))


def test_same_bits_twice_on_another_stream_and_in_a_graph(paged):
    c = make_case("16/8x128", 16, 1024, [70, 1, 300, 20] * 4, [1, 1, 3, 20] * 4, seed=9)
    first = call(paged, c)
    compare(c, first)
    assert torch.equal(first, call(paged, c))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(paged, c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    a, b = torch.empty_like(first), torch.empty_like(first)
    d = make_case("16/8x128", 16, 1024, [71, 2, 299, 19] * 4, [1, 1, 3, 20] * 4, seed=10)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        call(paged, c, out=a)
    with torch.cuda.graph(gb):
        call(paged, d, out=b)
    for _ in range(3):
        ga.replay()
        gb.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, first)
    compare(d, b)
    c["kv"].sub_(1)                                                # a replay reads the lengths of its time
    ga.replay()
    torch.cuda.synchronize()
    c["own"] = [n - 1 for n in c["own"]]
    compare(c, a)


@pytest.mark.parametrize("heads,own,new", [("16/16x128", [400, 1, 610, 77], [400, 1, 610, 77]), ("32/8x64", [900, 40, 410], [900, 3, 400]),
                                           ("16/8x128", [700, 650, 5], [700, 640, 5])])
def test_large_calls(paged, heads, own, new):
    """Calls whose rows' parts are added by fewer threads than the others': rows with one part, two, several and none."""
    c = make_case(heads, 32, 512, own, new, seed=19, pad=5)
    rows, H, D = c["q"].shape
    lse = torch.full((rows, H), 7.0, device="cuda:0")
    out = torch.full_like(c["q"], 3.0)
    call(paged, c, out=out, lse=lse)
    compare(c, out, lse)
    assert (out[-5:] == 3.0).all() and (lse[-5:] == 7.0).all()
    c["kv"] = ints([0, *c["kv"].tolist()[1:]])                     # the first request's rows see nothing
    call(paged, c, out=out, lse=lse)
    assert (out[:new[0]] == 0).all() and torch.isinf(lse[:new[0]]).all()
    c["own"] = [-512, *own[1:]]
    compare(c, out, lse)
    call(paged, dict(c, cu=ints([0, rows, 0, rows] + [0] * (len(own) - 3))), out=out, lse=lse)
    assert torch.isnan(out.float()).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("heads,prefix,own,new", [("32/8x64", 4096, [40, 60, 33, 90, 300], [40, 60, 33, 85, 1]),
                                                  ("16/8x128", 8192, [70, 100, 64, 20], [70, 90, 64, 3]),
                                                  ("5/1x128", 8192, [30, 75, 102], [30, 75, 102])])
def test_short_pieces_behind_a_long_prefix(paged, heads, prefix, own, new):
    """Requests of 128..511 rows, most of whose keys are the prefix: they share units and have strips of their own."""
    c = make_case(heads, 64, prefix, own, new, seed=21, pad=2)
    lse = torch.empty(c["q"].shape[0], c["q"].shape[1], device="cuda:0")
    compare(c, call(paged, c, lse=lse), lse)


def test_offsets_that_do_not_ascend_are_refused_on_the_device(paged):
    """cu_tokens that give a row to two requests or to none: every row becomes NaN, nothing outside the outputs is touched, and the
    next call on the same workspace is right."""
    for heads in ("32/8x64", "16/8x128"):
        c = make_case(heads, 16, 64, [40, 30, 9, 17], [1, 20, 2, 1], seed=14, pad=2)
        rows, H, D = c["q"].shape
        ws = paged.attention_workspace(c["q"], c["k"], 4, prefix_len=64)
        wide = torch.full((rows, H + 1, D), 5.0, dtype=torch.bfloat16, device="cuda:0")
        for cu in ([0, rows, 0, rows, 0], [0, 1, 21, 23, rows + 1], [1, 2, 21, 23, 24], [0, 21, 1, 23, 24], [-1, 1, 21, 23, 24],
                   [0, 1 << 30, 1 << 30, 1 << 30, (1 << 31) - 1]):
            lse = torch.zeros(rows, H, device="cuda:0")
            out = call(paged, dict(c, cu=ints(cu)), out=wide[:, :H], lse=lse, workspace=ws)
            assert torch.isnan(out.float()).all() and torch.isnan(lse).all(), cu
            assert (wide[:, H:] == 5.0).all()
        out = call(paged, c, workspace=ws)
        compare(c, out)
        assert (out[-2:] == 0).all()


def test_output_in_place_of_the_queries(paged):
    c = make_case("32/8x64", 16, 256, [40, 3, 200, 7, 150], [5, 3, 1, 7, 70], seed=15)
    want = call(paged, c)
    assert call(paged, c, out=c["q"]) is c["q"] and torch.equal(c["q"], want)


def test_two_calls_at_once_with_a_workspace_each(paged):
    a = make_case("16/8x128", 16, 1024, [70, 1, 300, 20] * 4, [1, 1, 3, 20] * 4, seed=9)
    b = make_case("32/8x64", 64, 2048, [33] * 24, [1] * 24, seed=16)
    want = [call(paged, c) for c in (a, b)]
    kept = [paged.attention_workspace(c["q"], c["k"], c["tables"].shape[0], prefix_len=c["prefix"]) for c in (a, b)]
    outs = [[torch.empty_like(c["q"]) for _ in range(8)] for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(8):
        for c, stream, ws, out in zip((a, b), streams, kept, outs):
            with torch.cuda.stream(stream):
                call(paged, c, out=out[i], workspace=ws)
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        assert all(torch.equal(w, o) for o in out)


def test_the_most_requests_and_no_rows(paged):
    # 1536 requests of one row each, some without any; a page named by several tables and twice in the prefix
    own = [1 + i % 23 for i in range(1536)]
    c = make_case("6/2x64", 16, 32, own, [0 if i % 7 == 3 else 1 for i in range(1536)], seed=17)
    c["prefix_table"] = ints([c["pool"][0]] * 2)
    t = c["tables"].tolist()
    for s in range(0, 1536, 5):
        t[s][2] = t[1][2]
        c["own"][s] = min(own[s], own[1])
    c["tables"], c["kv"] = ints(t), ints([32 + n for n in c["own"]])
    compare(c, call(paged, c))
    none = call(paged, dict(c, q=c["q"][:0]))
    assert none.shape == (0, 6, 64)


def test_pool_past_32_bit_offsets(paged):
    """Pages whose elements lie beyond 2^32 (and rows beyond 2^31 bytes) in a pool of 9 GB each for K and V."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    c = make_case("16/16x128", 64, 128, [130, 40], [1, 3], seed=18)
    n = c["k"].shape[0]
    big = (1 << 32) // (64 * 16 * 128) + 100
    for name in ("k", "v"):
        pool = torch.empty(big, 64, 16, 128, dtype=torch.bfloat16, device="cuda:0")
        pool[big - n:] = c[name]
        c[name] = pool
    c["tables"] = c["tables"] + (big - n) * ((c["tables"] >= 0) & (c["tables"] < n)).int()
    c["prefix_table"] = c["prefix_table"] + (big - n)
    compare(c, call(paged, c))


def test_tables_slots_and_attention_together(paged):
    """Admission, a step of prompt pieces and two decode steps as a server runs them, K and V rows stored through the slot map."""
    page, H, HK, D = 32, 16, 8, 128
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda:0").to(torch.bfloat16)
    prompts, prefix, pages = [40, 1, 100, 7], 96, 64
    k, v = rnd(pages, page, HK, D), rnd(pages, page, HK, D)
    order = torch.randperm(pages, generator=gen, device="cuda:0").to(torch.int32)
    shared, free = order[:3].contiguous(), order[3:].contiguous()
    tables = paged.build_block_tables(ints([prefix + n + 2 for n in prompts]), free, page_size=page, max_pages=9,
                                      prefix_table=shared)
    kv = torch.full((4,), prefix, dtype=torch.int32, device="cuda:0")
    dense = [[(k[shared.long()].reshape(-1, HK, D), v[shared.long()].reshape(-1, HK, D))] for _ in prompts]
    held = [prefix] * 4
    for new in (prompts, [1, 1, 0, 1], [1, 1, 1, 0]):
        T = sum(new) + 3
        step = paged.build_slot_map(tables.tables, kv, ints(new), page_size=page, tokens=T)
        kn, vn, q = rnd(T, HK, D), rnd(T, HK, D), rnd(T, H, D)
        rows = step.slots[step.active.bool()]
        assert rows.numel() == sum(new)
        k.view(-1, HK, D)[rows] = kn[step.active.bool()]
        v.view(-1, HK, D)[rows] = vn[step.active.bool()]
        out = paged.prefix_attention(q, k, v, tables.tables, step.kv_lengths, step.cu_tokens, prefix_table=shared,
                                     prefix_len=prefix)
        at = 0
        for s, n in enumerate(new):
            dense[s].append((kn[at:at + n], vn[at:at + n]))
            held[s] += n
            ks = torch.cat([x for x, _ in dense[s]]).double()
            vs = torch.cat([x for _, x in dense[s]]).double()
            for i in range(n):
                lim = held[s] - n + i + 1
                x = torch.einsum("hgd,khd->hgk", q[at + i].double().view(HK, 2, D), ks[:lim]) / math.sqrt(D)
                p = torch.softmax(x, -1)
                o = torch.einsum("hgk,khd->hgd", p, vs[:lim]).reshape(H, D)
                A = torch.einsum("hgk,khd->hgd", p, vs[:lim].abs()).reshape(H, D)
                assert ((out[at + i].double() - o).abs() <= 2.0 ** -8 * o.abs() + 2.0 ** -7.9 * A).all()
            at += n
        kv = step.kv_lengths
        assert (out[at:] == 0).all()


# ------------------------------------------------------------------------------------------------ NaN and infinity in sight
def compare_nonfinite(c, out, lse):
    """A row is NaN where the definition is, and only there; the others are within the derived tolerance."""
    o, want_lse, A, r = definition(c)
    real = c["cu_list"][-1]
    o, want_lse, A, r, out, lse = (x[:real] for x in (o, want_lse, A, r, out, lse))
    none = torch.isnan(o)
    assert torch.equal(torch.isnan(out), none), "rows that are NaN differ from the definition's"
    row = none[..., 0]
    assert torch.equal(torch.isnan(lse), row)
    err, tol = (out.double() - o).abs(), 2.0 ** -8 * o.abs() + (2.0 ** -8 + r) * (1 + 2.0 ** -6) * A
    assert (err <= tol)[~none].all()
    gap, slack = (lse.double() - want_lse).abs(), r[..., 0] + 2.0 ** -22 * want_lse.abs()
    assert (gap <= slack)[~row & ~torch.isinf(want_lse)].all()
    return row


def put_key(c, s, key, head, value):
    """K row of position `key` as request s sees it (None: any), in KV head `head`."""
    page = c["page"]
    ids = c["prefix_table"] if key < c["prefix"] else c["tables"][s]
    c["k"][int(ids[key // page]), key % page, head] = value


@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128"])
@pytest.mark.parametrize("at", [0, 72, 1024 + 64, 1024 + 104, 2048 - 64, 2048 - 8])
def test_nan_key_in_the_prefix(paged, heads, at):
    """A NaN in K of KV head h at the place h modulo 8 of a step of the shared prefix (the first step of a run of blocks and later
    ones): every row is NaN, whichever place it was."""
    few = make_case(heads, 16, 2048, [20, 5], [1, 3], seed=30)
    many = make_case(heads, 16, 2048, [9] * 60, [5] * 60, seed=31)       # two tiles a unit
    for c in (few, many):
        for head in range(8):
            put_key(c, None, at + head, head, float("nan"))
        lse = torch.empty(c["q"].shape[:2], device="cuda:0")
        row = compare_nonfinite(c, call(paged, c, lse=lse), lse)
        assert row.all()


@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128"])
@pytest.mark.parametrize("at", [8, 64 + 16, 256 + 24, 256 + 600])
def test_nan_key_in_a_long_piece(paged, heads, at):
    """The same in a piece of rows that are causal among themselves: rows before the key do not see it."""
    for prefix in (0, 256):
        c = make_case(heads, 32, prefix, [900, 3], [900, 1], seed=32)
        for head in range(8):
            put_key(c, 0, prefix + at + head, head, float("nan"))
        lse = torch.empty(c["q"].shape[:2], device="cuda:0")
        row = compare_nonfinite(c, call(paged, c, lse=lse), lse)
        assert row.any() and not row.all()


@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128"])
def test_infinite_scores_in_sight(paged, heads):
    """Keys with an infinity in one dimension: a score of plus infinity makes the row NaN, one of minus infinity counts as absent."""
    c = make_case(heads, 32, 512, [300, 40, 7], [1, 40, 300 // 60], seed=33)
    for head in range(8):
        for s, key in ((None, 200 + head), (None, 64 * 3 + 8 + head), (0, 512 + 33 + head), (1, 512 + 20)):
            put_key(c, s, key, head, 0.0)
            page = c["page"]
            ids = c["prefix_table"] if key < c["prefix"] else c["tables"][s]
            c["k"][int(ids[key // page]), key % page, head, head] = float("inf") if key % 2 else float("-inf")
    lse = torch.empty(c["q"].shape[:2], device="cuda:0")
    o, want, A, r = definition(c)
    out = call(paged, c, lse=lse)
    real = c["cu_list"][-1]
    none = torch.isnan(o)
    assert torch.equal(torch.isnan(out)[:real], none[:real]) and none[:real].any() and not none[:real].all()
    err, tol = (out.double() - o).abs(), 2.0 ** -8 * o.abs() + (2.0 ** -8 + r) * (1 + 2.0 ** -6) * A
    assert (err <= tol)[:real][~none[:real]].all()
    assert torch.equal(torch.isnan(lse)[:real], none[:real, :, 0])


@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128", "6/2x64", "5/1x128"])
@pytest.mark.parametrize("prefix", [0, 256])
def test_nan_key_behind_the_prefix(paged, heads, prefix):
    """A NaN in K of what a request holds behind the prefix: its only key, the only one of a piece, one among others.  The rows of
    the request that see it are NaN in that KV head, and no others are."""
    HK = HEADS[heads][1]
    for own, new, s, key in (([1], [1], 0, 0), ([1, 7], [1, 1], 0, 0), ([33, 2], [1, 1], 0, 32), ([65, 40], [3, 1], 0, 64),
                             ([40, 100], [1, 5], 1, 96), ([40, 100], [1, 5], 1, 17), ([20] * 30, [2] * 30, 11, 5)):
        for head in {0, HK - 1}:
            c = make_case(heads, 16, prefix, own, new, seed=34)
            put_key(c, s, prefix + key, head, float("nan"))
            lse = torch.empty(c["q"].shape[:2], device="cuda:0")
            row = compare_nonfinite(c, call(paged, c, lse=lse), lse)
            assert row.any()


@pytest.mark.parametrize("heads", ["32/8x64", "16/16x128"])
@pytest.mark.parametrize("prefix", [0, 512])
def test_nan_key_behind_the_prefix_in_a_large_call(paged, heads, prefix):
    """The same where the parts are added by fewer threads (more than 888 rows)."""
    own, new = [920, 1, 40, 33, 2], [920, 1, 3, 1, 2]
    for s, key in ((1, 0), (2, 39), (3, 32), (4, 1)):
        c = make_case(heads, 32, prefix, own, new, seed=35)
        put_key(c, s, prefix + key, 3 if heads == "32/8x64" else 0, float("nan"))
        lse = torch.empty(c["q"].shape[:2], device="cuda:0")
        row = compare_nonfinite(c, call(paged, c, lse=lse), lse)
        assert row.any() and not row[:920].any()


def test_outputs_beside_the_inputs_and_over_them(paged):
    """Outputs that lie right beside their inputs are taken, those that cover part of one are refused and nothing is written."""
    from qimeng_megakernel_b200 import _lib
    want = paged.build_slot_map(ints([[3, 4]] * 3), ints([1, 20, 5]), ints([2, 1, 1]), page_size=16, tokens=5)
    buf = torch.full((16,), -5, dtype=torch.int32, device="cuda:0")
    kv, new = buf[3:6], buf[6:9]
    kv.copy_(ints([1, 20, 5]))
    new.copy_(ints([2, 1, 1]))
    out = paged.SlotMap.empty(3, 5, "cuda:0")
    out.kv_lengths, out.cu_tokens = buf[:3], buf[9:13]
    paged.build_slot_map(ints([[3, 4]] * 3), kv, new, page_size=16, tokens=5, out=out)
    for name in ("slots", "positions", "seq_ids", "active", "cu_tokens", "kv_lengths"):
        assert torch.equal(getattr(out, name), getattr(want, name)), name
    before = buf.clone()
    for name, t in (("kv_lengths", buf[1:4]), ("kv_lengths", buf[7:10]), ("cu_tokens", buf[5:9])):
        bad = paged.SlotMap.empty(3, 5, "cuda:0")
        setattr(bad, name, t)
        with pytest.raises(_lib.QmkError, match="overlaps"):
            paged.build_slot_map(ints([[3, 4]] * 3), kv, new, page_size=16, tokens=5, out=bad)
    tables = paged.BlockTables(buf[:6].view(3, 2), buf[14:])
    with pytest.raises(_lib.QmkError, match="tables overlaps lengths"):
        paged.build_block_tables(kv, new, page_size=16, max_pages=2, out=tables)
    assert torch.equal(buf, before)


def test_refusals_say_why(paged):
    """Calls inside the limits of every single argument that are refused all the same name the reason."""
    from qimeng_megakernel_b200 import _lib
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda:0")
    pool = z(2, 256, 8, 64)
    q, tables = z(16384, 32, 64), z(1536, 4096, t=torch.int32)
    args = (q, pool, pool, tables, z(1536, t=torch.int32), z(1537, t=torch.int32))
    with pytest.raises(_lib.QmkError, match="32 bits"):
        paged.prefix_attention(*args)
    paged.prefix_attention(*args[:3], tables[:, :3400].contiguous(), *args[4:])
    few = (z(2, 32, 64), pool, pool, z(1, 4, t=torch.int32), z(1, t=torch.int32), z(2, t=torch.int32))
    ws = paged.attention_workspace(few[0], pool, 1)
    with pytest.raises(_lib.QmkError, match="workspace"):
        paged.prefix_attention(*few, workspace=torch.empty(ws.numel() + 16, dtype=torch.uint8, device="cuda:0")[16:])
    odd = z(pool.numel() + 4)[4:].view(pool.shape)
    with pytest.raises(_lib.QmkError, match="pages"):
        paged.prefix_attention(few[0], odd, odd, *few[3:])
    with pytest.raises(ValueError, match="1024 query heads"):
        paged.prefix_attention(z(2, 1040, 64), z(2, 16, 65, 64), z(2, 16, 65, 64), *few[3:])


@pytest.mark.parametrize("rows,seqs,most", [(8192, 1, 110e6), (8192, 4, 125e6), (64, 64, 60e6)])
def test_workspace_has_room_for_short_requests_only_as_far_as_there_can_be_any(paged, rows, seqs, most):
    """A request of 512 (token, head) rows and more has no strips: one piece of 8192 rows needs records for 511 short ones at most."""
    q = torch.empty(rows, 16, 128, dtype=torch.bfloat16, device="cuda:0")
    assert paged.attention_workspace(q, torch.empty(1, 16, 16, 128, dtype=torch.bfloat16, device="cuda:0"), seqs).numel() < most


@pytest.mark.parametrize("heads", ["32/8x64", "16/8x128"])
def test_rows_of_minus_infinity_alone_see_nothing(paged, heads):
    """Keys of minus infinity count as absent, and a row that has no others gives zeros and an lse of minus infinity: a single own
    key, a whole short request, the first rows of a long piece."""
    c = make_case(heads, 16, 0, [1, 40, 300], [1, 3, 300], seed=36)
    c["q"] = c["q"].abs() + 1
    for s, keys in ((0, range(1)), (1, range(40)), (2, range(70))):
        for key in keys:
            c["k"][int(c["tables"][s, key // 16]), key % 16] = float("-inf")
    lse = torch.empty(c["q"].shape[:2], device="cuda:0")
    out = call(paged, c, lse=lse)
    o, want, A, r = definition(c)
    assert torch.isinf(want[:74]).all() and not torch.isinf(want[74:]).any()
    assert (out[:74] == 0).all() and (lse[:74] == float("-inf")).all()
    err, tol = (out.double() - o).abs(), 2.0 ** -8 * o.abs() + (2.0 ** -8 + r) * (1 + 2.0 ** -6) * A
    assert (err <= tol)[74:].all()
