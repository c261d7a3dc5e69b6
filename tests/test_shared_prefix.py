"""plan_shared_prefix and shared_prefix_decode_attention against a plain plan
and against attention in 64 bits over the whole table, with their refusals.

Tolerance of the attention, from the arithmetic: a weight w_t / sum w differs
from the exact one by a relative e_w = 2^-8 (its rounding to bf16; the sum is of
the rounded weights) + the scores' fp32 error, so an output by at most
e_w sum_t p_t |v_t - o|; fp32 accumulation adds T 2^-24 sum_t p_t |v_t| and the
result's rounding 2^-8 |o|.  With queries of zero every weight is exactly one,
and the first term falls away: those cases see a single wrong token."""
import math
import random

import numpy as np
import pytest
import torch

import workloads as W
from vortex_torch import _hip
from vortex_torch.decode_attention import SharedPrefixPlan, plan_shared_prefix, shared_prefix_decode_attention


# ------------------------------------------------------------------- tables
def _table(groups, P, H, seed, scrambled_heads=False):
    """groups: (shared pages, [own tokens of each request]); own tokens None: an
    empty request.  Returns (indptr, indices, last, pool pages); every entry is
    page * H + h."""
    r = random.Random(seed)
    total = sum(s + sum(-(-t // P) for t in own if t) for s, own in groups) + 5
    free = list(range(total))
    r.shuffle(free)
    indptr, indices, last = [0], [], []
    for shared, own in groups:
        pages = [free.pop() for _ in range(shared)]
        for t in own:
            mine = pages + [free.pop() for _ in range(-(-t // P))] if t else []
            for h in range(H):
                # (scrambled: each head's own order, as in a table of selected pages)
                order = sorted(mine, key=lambda p: (p * 7 + h * 13) % 31) if scrambled_heads else mine
                indices += [p * H + h for p in order]
                indptr.append(len(indices))
                last.append((t - 1) % P + 1 if t else 0)
    return (torch.tensor(indptr, dtype=torch.int32), torch.tensor(indices, dtype=torch.int32),
            torch.tensor(last, dtype=torch.int32), total)


def _plain_plan(indptr, indices, B, H, ids=None):
    leaders, shared = [0] * (B * H), [0] * (B * H)
    rows = [indices[indptr[s]:indptr[s + 1]].tolist() for s in range(B * H)]
    for h in range(H):
        b = 0
        while b < B:
            run = [b]
            while b + 1 < B and rows[b * H + h] and rows[(b + 1) * H + h] and (
                    ids[b] == ids[b + 1] if ids is not None else rows[b * H + h][0] == rows[(b + 1) * H + h][0]):
                b += 1
                run.append(b)
            common = 0
            if len(run) > 1:
                mine = [rows[x * H + h] for x in run]
                most = min(len(x) for x in mine) - 1
                while common < most and len({x[common] for x in mine}) == 1:
                    common += 1
            for x in run:
                leaders[x * H + h], shared[x * H + h] = run[0], common
            b += 1
    return leaders, shared


PLANS = {
    "one_run": ([(9, [5, 17, 40])], 16, 2),
    "alone": ([(0, [100]), (0, [1])], 16, 3),
    "one_request": ([(4, [3])], 16, 1),
    "empty_splits_run": ([(6, [20, 20, None, 20, 20]), (0, [None, None])], 16, 2),
    "many_runs": ([(3, [7] * 8)] * 20 + [(0, [50])] * 3 + [(40, [1, 2])], 16, 4),
    "page_of_one": ([(700, [1, 2, 3]), (5, [1])], 1, 2),
    "long": ([(5000, [1, 300]), (2100, [16] * 5)], 16, 1),
    "shared_of_one_page": ([(1, [1, 1])], 64, 8),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", PLANS)
@pytest.mark.parametrize("scrambled", [False, True])
def test_plan_finds_what_is_shared(gpu, name, scrambled):
    groups, P, H = PLANS[name]
    indptr, indices, _, _ = _table(groups, P, H, 3, scrambled)
    B = (indptr.numel() - 1) // H
    ids = torch.tensor([b // 3 for b in range(B)], dtype=torch.int32)
    for g in (None, ids, torch.zeros_like(ids)):
        plan = plan_shared_prefix(indptr.to(gpu), indices.to(gpu), B, H, 2, 128, P,
                                  group_ids=None if g is None else g.to(gpu))
        leaders, shared = _plain_plan(indptr, indices, B, H, None if g is None else g.tolist())
        assert plan.leaders.tolist() == leaders and plan.shared_pages.tolist() == shared


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_plan_of_random_tables(gpu, seed):
    r = random.Random(seed)
    P, H = r.choice([1, 16, 64]), r.choice([1, 3, 8])
    groups = [(r.choice([0, 1, 7, 300]), [r.choice([1, 30, 200, None]) for _ in range(r.randint(1, 9))])
              for _ in range(r.choice([1, 12, 150]))]
    indptr, indices, _, _ = _table(groups, P, H, seed)
    B = (indptr.numel() - 1) // H
    plan = plan_shared_prefix(indptr.to(gpu), indices.to(gpu), B, H, 1, 64, P)
    leaders, shared = _plain_plan(indptr, indices, B, H)
    assert plan.leaders.tolist() == leaders and plan.shared_pages.tolist() == shared


@pytest.mark.gpu
def test_plan_entries_outside_the_table(gpu):
    """Segments whose range leaves kv_indices, or runs backwards, count as empty."""
    indptr, indices, _, _ = _table([(4, [20, 20, 20, 20])], 16, 1, 1)
    bad = indptr.clone()
    bad[4] = indices.numel() + 7
    plan = plan_shared_prefix(bad.to(gpu), indices.to(gpu), 4, 1, 1, 64, 16)
    assert plan.leaders.tolist() == [0, 0, 0, 3] and plan.shared_pages.tolist() == [4, 4, 4, 0]
    bad = indptr.clone()
    bad[1] = -5
    plan = plan_shared_prefix(bad.to(gpu), indices.to(gpu), 4, 1, 1, 64, 16)
    assert plan.leaders.tolist() == [0, 1, 2, 2] and plan.shared_pages.tolist() == [0, 0, 4, 4]


# ---------------------------------------------------------------- attention
def _exact(q, k, v, indptr, indices, last, scale):
    """(outputs, tolerance) of every query row in 64 bits; entries outside the
    pool are masked, a segment without tokens gives zeros."""
    S, P, D = indptr.numel() - 1, k.shape[1], k.shape[2]
    q = q.view(S, -1, D).double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    ptr, ll = indptr.tolist(), last.tolist()
    for s in range(S):
        rows = indices[ptr[s]:ptr[s + 1]].long()
        n = (rows.numel() - 1) * P + ll[s]
        if rows.numel() == 0 or n <= 0:
            continue
        ok = ((rows >= 0) & (rows < k.shape[0])).repeat_interleave(P)[:n]
        rows = rows.clamp(0, k.shape[0] - 1)
        kk, vv = (t[rows].reshape(-1, D)[:n][ok].double() for t in (k, v))
        if kk.shape[0] == 0:
            continue
        sc = q[s] @ kk.t().contiguous() * scale
        p = torch.softmax(sc, -1)
        o = p @ vv
        size = (q[s].abs() @ kk.abs().t().contiguous()).amax(-1, keepdim=True) * abs(scale)
        # D products and sums, the scale, the exponent's argument and 2^x, at numerator and denominator
        e_s = 2 * (D + 8) * 2.0 ** -24 * size + 2.0 ** -22
        exact_weights = (q[s].abs().amax(-1, keepdim=True) == 0) | (scale == 0)
        e_w = torch.where(exact_weights, 0.0, 1.01 * 2.0 ** -8 + e_s)
        if vv.shape[0] * D * q.shape[1] < 1 << 25:
            spread = torch.einsum("gt,gtd->gd", p, (vv[None] - o[:, None]).abs())
        else:  # (a bound of it)
            spread = p @ vv.abs() + o.abs()
        out[s] = o
        bound[s] = e_w * spread + (n + 64) * 2.0 ** -24 * (p @ vv.abs()) + 2.0 ** -8 * o.abs() * 1.01 + 1e-37
    return out.view(-1, D), bound.view(-1, D)


def _inputs(table, P, H, G, D, seed, device, std=1.5):
    indptr, indices, last, pages = table
    gen = torch.Generator().manual_seed(seed)
    S = indptr.numel() - 1
    q = (torch.randn((S, G, D), generator=gen) * std).bfloat16().to(device)
    k, v = (torch.randn((pages * H, P, D), generator=gen).bfloat16().to(device) for _ in range(2))
    # slots that hold no token are anything, NaN and infinities too
    used = torch.zeros((pages * H, P), dtype=torch.bool)
    for s in range(S):
        rows = indices[indptr[s]:indptr[s + 1]].tolist()
        for i, row in enumerate(rows):
            if 0 <= row < pages * H:
                used[row, :P if i + 1 < len(rows) else int(last[s])] = True
    for t, poison in ((k, float("nan")), (v, float("inf"))):
        t[~used.to(device)] = poison
    return q, k, v


def _attention(table, P, H, G, D, device, seed=0, scale=None, zero_queries=False, ids=None):
    indptr, indices, last, _ = table
    q, k, v = _inputs(table, P, H, G, D, seed, device)
    if zero_queries:
        q.zero_()
    B = (indptr.numel() - 1) // H
    t = [x.to(device) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], B, H, G, D, P, group_ids=ids)
    out = torch.full((B * H * G + 2, D), 5.0, dtype=torch.bfloat16, device=device)
    got = shared_prefix_decode_attention(q, k, v, *t, plan, sm_scale=scale, out=out[1:-1].view(B * H, G, D))
    want, bound = _exact(q, k, v, indptr, t[1], last, 1 / math.sqrt(D) if scale is None else scale)
    err = (got.view(-1, D).double() - want).abs()
    assert bool((err <= bound).all()), f"off by up to {float((err / bound.clamp(min=1e-30)).max()):.2f} of the bound"
    assert bool((out[0] == 5).all()) and bool((out[-1] == 5).all())
    return got


TABLES = {
    # one token of its own each, just past the shared pages
    "ones": ([(20, [1, 1, 1])], 16),
    # rows of one tile (up to 32), two (up to 64), all four waves, and several tiles, by group size
    "few": ([(30, [40, 3, 77, 16])], 16),
    "seven": ([(17, [5, 100, 1, 16, 33, 250, 64])], 16),
    "twenty": ([(40, [9 + 11 * i for i in range(20)])], 16),
    "forty": ([(12, [1 + 7 * i for i in range(40)])], 16),
    # nothing shared, nothing to share, next to a run, empty requests between
    "mixed": ([(0, [300]), (9, [20, 20]), (0, [1]), (30, [2, None, 90, 5]), (0, [None]), (16, [600, 1])], 16),
    "all_empty": ([(0, [None, None])], 16),
    # shared stretches too short to be read once
    "short": ([(2, [30, 50]), (1, [1, 1, 1]), (7, [16] * 4)], 16),
    # other pages: of one token, not a power of two, large; chunks end inside a tile
    "page1": ([(333, [1, 50, 2]), (0, [129])], 1),
    "page24": ([(13, [24, 25, 23]), (0, [100])], 24),
    "page64": ([(9, [64, 1, 200, 63, 65])], 64),
    # longer than one chunk per item, uneven
    "long": ([(300, [1, 700]), (0, [3000])], 16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("name", TABLES)
def test_attention_over_tables(gpu, name, D):
    groups, P = TABLES[name]
    for H, G in ((1, 1), (2, 2), (1, 5), (2, 8)):
        table = _table(groups, P, H, 5)
        _attention(table, P, H, G, D, gpu, seed=G)
        _attention(table, P, H, G, D, gpu, seed=G, zero_queries=True)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 1e-3, 40.0])
def test_attention_scales(gpu, scale):
    _attention(_table([(24, [60, 1, 200])], 16, 2, 1), 16, 2, 4, 128, gpu, scale=scale)


@pytest.mark.gpu
def test_attention_large_run_and_table(gpu):
    _attention(_table([(64, [1 + 5 * i for i in range(70)])], 16, 1, 2), 16, 1, 8, 128, gpu)
    _attention(_table([(40, [30] * 8)] * 24, 16, 8, 2), 16, 8, 2, 128, gpu)
    _attention(_table([(1200, [100, 20000])], 16, 1, 2), 16, 1, 4, 128, gpu)


@pytest.mark.gpu
def test_attention_ids_and_selected_pages(gpu):
    """Groups that the caller names (one of them of requests that share
    nothing), and a table whose heads hold other pages each."""
    table = _table([(20, [30, 40, 50, 60]), (0, [70]), (0, [80])], 16, 2, 9)
    for ids in ([0, 0, 1, 1, 2, 2], [0] * 6, [0, 1, 2, 3, 4, 5], [-1, -1, 7, 7, 7, 7]):
        _attention(table, 16, 2, 4, 128, gpu, ids=torch.tensor(ids, dtype=torch.int32, device=gpu))
    _attention(_table([(20, [30, 40, 50, 60])], 16, 4, 9, scrambled_heads=True), 16, 4, 2, 128, gpu)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_attention_entries_outside_the_pool(gpu, D):
    """Pages that do not exist are masked, in shared and in own pages; a request
    of nothing else gives zeros."""
    indptr, indices, last, pages = _table([(20, [40, 70, 30]), (0, [33])], 16, 2, 4)
    rows = pages * 2
    for s in range(6):  # the same entries of every request, and one of its own
        for i, bad in ((0, -1), (3, rows), (19, 2 ** 31 - 1), (21, -2 ** 31)):
            indices[indptr[s] + i] = bad
    indices[indptr[6]:indptr[7]] = -1
    got = _attention((indptr, indices, last, pages), 16, 2, 4, D, gpu)
    assert int(got.view(8, 4, D)[6].count_nonzero()) == 0


@pytest.mark.gpu
def test_attention_nan_scores_give_nan(gpu):
    """A key of NaN at a token that counts reaches every result of its segment, and no other."""
    indptr, indices, last, _ = table = _table([(20, [40, 70]), (0, [50])], 16, 1, 4)
    q, k, v = _inputs(table, 16, 1, 2, 128, 0, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    k[indices[0], 3] = float("nan")
    plan = plan_shared_prefix(t[0], t[1], 3, 1, 2, 128, 16)
    nan = shared_prefix_decode_attention(q, k, v, *t, plan).isnan()
    assert bool(nan[:2].all()) and not bool(nan[2].any())


# (shared pages, own tokens): a request's only own token next to longer ones; workgroups of four
# short requests; nothing shared, finished where they are or joined; several row tiles; four-wave joins
NAN_TABLES = {
    "few": [(20, [1, 40, 1])],
    "many": [(20, [1] * 90)],
    "alone": [(0, [1]), (0, [5])],
    "many_alone": [(0, [1])] * 90,
    "rows": [(12, [1 + 7 * (i % 5) for i in range(40)])],
    "long": [(1200, [1, 9000])],
}


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("name", NAN_TABLES)
def test_attention_keeps_nan_where_nothing_else_is_seen(gpu, name, D):
    """A query of NaN, and a NaN key that is all a request holds of its own or
    all it holds at all, give NaN in just the rows that see them, whatever way
    the tokens are divided; all other rows keep their bits."""
    H, G, P = (1, 2, 16) if name == "long" else (8, 2, 16)
    indptr, indices, last, _ = table = _table(NAN_TABLES[name], P, H, 5)
    q, k, v = _inputs(table, P, H, G, D, 0, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    B = (indptr.numel() - 1) // H
    plan = plan_shared_prefix(t[0], t[1], B, H, G, D, P)
    clean = shared_prefix_decode_attention(q, k, v, *t, plan)
    assert not bool(clean.isnan().any())

    def check(q, k, rows):
        got = shared_prefix_decode_attention(q, k, v, *t, plan)
        assert bool(got[rows].isnan().all())
        assert torch.equal(got[~rows], clean[~rows])

    none = torch.zeros((B * H, G), dtype=torch.bool, device=gpu)
    turned, rows = q.clone(), none.clone()
    turned[0, 1] = turned[-1, 0] = float("nan")
    rows[0, 1] = rows[-1, 0] = True
    check(turned, k, rows)
    keys, rows = k.clone(), none.clone()
    keys[indices[indptr[1] - 1], 0] = float("nan")  # the first token that segment 0 does not share
    rows[0] = True
    check(q, keys, rows)
    shared = int(plan.shared_pages[0])
    keys, rows = k.clone(), none.clone()
    keys[indices[indptr[0]:indptr[1]].long()] = float("nan")  # all of segment 0's, and who shares them
    rows[0] = True
    if shared:
        rows[::H] = plan.leaders.view(B, H)[:, :1] == 0
    check(q, keys, rows)


@pytest.mark.gpu
def test_attention_follows_last_page_lengths(gpu):
    """kv_last_page_len may change after the plan."""
    indptr, indices, last, _ = table = _table([(30, [40, 3, 77, 16])], 16, 2, 7)
    q, k, v = _inputs(table, 16, 2, 2, 128, 0, gpu)
    k.nan_to_num_(0.5)
    v.nan_to_num_(0.5, 0.5, 0.5)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], 4, 2, 2, 128, 16)
    for ll in (1, 9, 16, 0, -3, 99):
        t[2].fill_(ll)
        got = shared_prefix_decode_attention(q, k, v, *t, plan)
        want, bound = _exact(q, k, v, indptr, t[1], t[2].clamp(0, 16), 128 ** -0.5)
        assert bool(((got.view(-1, 128).double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,requests,G", [(128, 2, 4), (64, 10, 4), (128, 20, 8), (256, 3, 8), (256, 12, 4)])
def test_attention_pool_past_32_bits(gpu, D, requests, G):
    """Pages at the end of pools of over 2^32 bytes, by rows of one tile and of several."""
    P, shared = 16, 30
    pages = (1 << 32) // (P * D * 2) + shared + requests
    k, v = (torch.zeros((pages, P, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    last_pages = shared + requests
    k[-last_pages:].normal_()
    v[-last_pages:].normal_()
    k[:last_pages] = float("nan")
    rows = torch.arange(pages - last_pages, pages, dtype=torch.int32)
    indices = torch.cat([torch.cat([rows[:shared], rows[shared + i:shared + i + 1]]) for i in range(requests)])
    indptr = torch.arange(requests + 1, dtype=torch.int32) * (shared + 1)
    last = torch.tensor([1 + (5 * i) % P for i in range(requests)], dtype=torch.int32)
    q = torch.randn((requests, G, D), dtype=torch.bfloat16, device=gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], requests, 1, G, D, P)
    assert plan.shared_pages.tolist() == [shared] * requests
    got = shared_prefix_decode_attention(q, k, v, *t, plan)
    want, bound = _exact(q, k, v, indptr, t[1], last, D ** -0.5)
    assert bool(((got.view(-1, D).double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,requests,G", [(128, 2, 4), (64, 20, 8), (128, 20, 8), (256, 12, 4)])
def test_attention_pool_past_31_bits(gpu, D, requests, G):
    """Pages at the end of pools of 3.5 GiB, which 32 bits of offset still reach."""
    P, shared = 16, 30
    pages = (7 << 29) // (P * D * 2)
    mine = shared + requests
    k, v = (torch.zeros((pages, P, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    k[-mine:].normal_()
    v[-mine:].normal_()
    k[:mine] = float("nan")
    rows = torch.arange(pages - mine, pages, dtype=torch.int32)
    indices = torch.cat([torch.cat([rows[:shared], rows[shared + i:shared + i + 1]]) for i in range(requests)])
    indptr = torch.arange(requests + 1, dtype=torch.int32) * (shared + 1)
    last = torch.tensor([1 + (5 * i) % P for i in range(requests)], dtype=torch.int32)
    q = torch.randn((requests, G, D), dtype=torch.bfloat16, device=gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], requests, 1, G, D, P)
    got = shared_prefix_decode_attention(q, k, v, *t, plan)
    want, bound = _exact(q, k, v, indptr, t[1], last, D ** -0.5)
    assert bool(((got.view(-1, D).double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("zero_queries", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_rows_of_many_partial_results(gpu, D, zero_queries):
    """More than 5120 / D of them each on average, which four waves join; the
    last batch of them is ragged, and one row's fewer than a batch."""
    _attention(_table([(1200, [100, 20000])], 16, 1, 2), 16, 1, 4, D, gpu, zero_queries=zero_queries)
    _attention(_table([(1500, [9000, 1, 4000]), (0, [40000])], 16, 1, 3), 16, 1, 1, D, gpu, zero_queries=zero_queries)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("name", ["few", "mixed", "long"])
def test_table_with_room_behind_it(gpu, name, D):
    """kv_indices as a server holds it, sized for the longest contexts: what lies
    behind the last segment is not read, and the plan finds the same."""
    groups, P = TABLES[name]
    H, G = 2, 2
    indptr, indices, last, pages = table = _table(groups, P, H, 5)
    B = (indptr.numel() - 1) // H
    q, k, v = _inputs(table, P, H, G, D, 1, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    wide = torch.full((B * H * 8192,), -7, dtype=torch.int32, device=gpu)
    wide[:indices.numel()] = t[1]
    plan = plan_shared_prefix(t[0], wide, B, H, G, D, P)
    leaders, shared = _plain_plan(indptr, indices, B, H)
    assert plan.leaders.tolist() == leaders and plan.shared_pages.tolist() == shared
    got = shared_prefix_decode_attention(q, k, v, t[0], wide, t[2], plan)
    want, bound = _exact(q, k, v, indptr, t[1], last, D ** -0.5)
    assert bool(((got.view(-1, D).double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_prefixes_behind_a_common_page(gpu):
    """Requests that all begin with one page and go on in groups: without ids
    they are one run and share that page alone; ids give each group its own."""
    H, G, D, P, longest = 2, 2, 128, 16, 40
    r = random.Random(4)
    sizes, own = [4, 1, 3, 2], 3  # requests of a group; pages of their own, at most
    free = list(range(1, 1 + len(sizes) * longest + sum(sizes) * own))
    r.shuffle(free)
    rows, ids, lengths = [], [], []
    for g, n in enumerate(sizes):
        body = [free.pop() for _ in range(longest - 7 * g)]
        lengths += [1 + len(body)] * n
        ids += [g] * n
        rows += [[0] + body + [free.pop() for _ in range(r.randint(1, own))] for _ in range(n)]
    B = len(rows)
    indices = torch.tensor([p * H + h for row in rows for h in range(H) for p in row], dtype=torch.int32)
    indptr = torch.tensor([0] + [len(row) for row in rows for _ in range(H)], dtype=torch.int32).cumsum(0).int()
    last = torch.tensor([r.randint(1, P) for _ in range(B)], dtype=torch.int32).repeat_interleave(H)
    table = indptr, indices, last, len(free) + sum(sizes) * own + len(sizes) * longest + 1
    t = [x.to(gpu) for x in (indptr, indices)]
    plan = plan_shared_prefix(*t, B, H, G, D, P)
    assert plan.leaders.tolist() == [0] * (B * H) and plan.shared_pages.tolist() == [1] * (B * H)
    named = torch.tensor(ids, dtype=torch.int32, device=gpu)
    plan = plan_shared_prefix(*t, B, H, G, D, P, group_ids=named)
    first = [ids.index(g) for g in ids]
    assert plan.leaders.view(B, H)[:, 0].tolist() == first == plan.leaders.view(B, H)[:, 1].tolist()
    want = [0 if sizes[g] == 1 else n for g, n in zip(ids, lengths)]
    assert plan.shared_pages.view(B, H)[:, 0].tolist() == want == plan.shared_pages.view(B, H)[:, 1].tolist()
    for g in (None, named):
        _attention(table, P, H, G, D, gpu, ids=g)
        _attention(table, P, H, G, D, gpu, ids=g, zero_queries=True)


# Short requests share workgroups where there are many: with a run's pages, without
# (finished where they are), next to long and empty ones, at a batch's ragged end.
MANY = {
    "behind_one": [(20, [1 + i % 17 for i in range(90)])],
    "alone": [(0, [1 + (37 * i) % 128]) for i in range(90)],
    "mixed": [(10, [3, None, 128, 129, 1]), (0, [None, None, None]), (0, [5]), (0, [1000]), (12, [1, 2])] * 9,
    "pairs": [(8, [16, 1]), (0, [None, 7, None, None])] * 15 + [(0, [9])],
}


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("name", MANY)
def test_attention_many_short_requests(gpu, name, D):
    _attention(_table(MANY[name], 16, 8, 3), 16, 8, 2, D, gpu)
    _attention(_table(MANY[name], 16, 8, 3), 16, 8, 1, D, gpu, zero_queries=True)
    _attention(_table(MANY[name], 8, 8, 3), 8, 8, 8, D, gpu)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [1, 3])
def test_plan_and_attention_of_thousands_of_requests(gpu, H):
    """More requests than the planner keeps in LDS."""
    r = random.Random(5)
    groups = [(r.choice([0, 1, 12]), [r.choice([1, 20, 40, None]) for _ in range(r.randint(1, 60))])
              for _ in range(100)]
    indptr, indices, last, pages = table = _table(groups, 16, H, 6)
    B = (indptr.numel() - 1) // H
    assert B > 2048
    plan = plan_shared_prefix(indptr.to(gpu), indices.to(gpu), B, H, 2, 64, 16)
    leaders, shared = _plain_plan(indptr, indices, B, H)
    assert plan.leaders.tolist() == leaders and plan.shared_pages.tolist() == shared
    _attention(table, 16, H, 2, 64, gpu)


@pytest.mark.gpu
def test_attention_takes_layout_tagged_tensors(gpu):
    """Pools and tables as a flow holds them (vTensors)."""
    from vortex_torch.abs import FORMAT, as_vtensor

    indptr, indices, last, _ = table = _table([(20, [40, 3, 77])], 16, 2, 7)
    q, k, v = _inputs(table, 16, 2, 2, 128, 0, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    want = shared_prefix_decode_attention(q, k, v, *t, plan_shared_prefix(t[0], t[1], 3, 2, 2, 128, 16))
    tagged = as_vtensor(t[1].view(-1, 1, 1), FORMAT.RAGGED)
    plan = plan_shared_prefix(t[0], tagged, 3, 2, 2, 128, 16)
    got = shared_prefix_decode_attention(as_vtensor(q, FORMAT.BATCHED), as_vtensor(k, FORMAT.PAGED),
                                         as_vtensor(v, FORMAT.PAGED), t[0], tagged, t[2], plan,
                                         out=torch.zeros_like(q))
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_attention_streams_and_repeats(gpu):
    """Calls on two streams at once with one plan, and repeats, agree bit for bit."""
    table = _table([(60, [30 + i for i in range(16)])], 16, 4, 7)
    indptr, indices, last, _ = table
    q, k, v = _inputs(table, 16, 4, 4, 128, 0, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], 16, 4, 4, 128, 16)
    first = shared_prefix_decode_attention(q, k, v, *t, plan)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(shared_prefix_decode_attention(q, k, v, *t, plan))
    torch.cuda.synchronize()
    assert all(torch.equal(first, g) for g in got)


def _step(ic, b, layers, positions, table, loc, plan, P, outs):
    """A decode step: tables, what they share, then layer by layer the new
    tokens rotated and stored, and attention over everything."""
    from vortex_torch.cache import set_kv_buffer_rope
    from vortex_torch.indexer.utils_sglang import plan_decode

    plan_decode(b.seq_lens, b.req_to_token, b.req_indices, ic)
    B, H, G, D, _ = plan.sizes
    plan_shared_prefix(ic.dense_kv_indptr, ic.dense_kv_indices, B, H, G, D, P, plan=plan)
    for (q, nk, nv, k, v), o in zip(layers, outs):
        turned = set_kv_buffer_rope(k, v, q, nk, nv, loc, P, positions, table)
        shared_prefix_decode_attention(turned, k, v, ic.dense_kv_indptr, ic.dense_kv_indices, ic.kv_last_page_len,
                                       plan, out=o)


@pytest.mark.gpu
def test_captured_decode_step(gpu):
    """plan_decode, plan_shared_prefix, set_kv_buffer_rope and the attention of
    two layers in one graph, replayed while the requests' lengths, and with them
    what they share, change; every replay equals the eager step bit for bit."""
    H, G, D, P, shared = 2, 4, 128, 16, 40
    most = [900, 700, 1200, 660, 800]
    pool = sum(-(-n // P) for n in most) + 3
    batch = W.make_batch(most, pool_pages=pool, seed=61, num_kv_heads=H, group_size=G, head_dim=D)
    first = batch.req_to_token[batch.req_indices[0], :shared * P].clone()
    for i in (1, 2, 4):  # requests 0, 1, 2 share their first pages, 4 does but has 3 before it
        batch.req_to_token[batch.req_indices[i], :shared * P] = first
    ic, _ = W.make_contexts(batch, gpu)
    b = batch.to(gpu)
    B = len(most)
    gen = torch.Generator().manual_seed(0)
    randn = lambda *s: torch.randn(s, generator=gen).bfloat16().to(gpu)  # noqa: E731
    layers = [(randn(B, H * G, D), randn(B, H, D), randn(B, H, D), randn(pool * H, P, D), randn(pool * H, P, D))
              for _ in range(2)]
    half = torch.arange(D // 2) / (D // 2)
    angle = torch.arange(2048)[:, None] * 1e4 ** -half
    table = torch.cat([angle.cos(), angle.sin()], 1).float().to(gpu)
    positions, loc = torch.zeros(B, dtype=torch.int64, device=gpu), torch.zeros(B, dtype=torch.int64, device=gpu)

    def at(lens):
        b.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        positions.copy_(torch.tensor([max(n - 1, 0) for n in lens]))
        loc.copy_(torch.tensor([int(batch.req_to_token[batch.req_indices[i], n - 1]) if n else -1
                                for i, n in enumerate(lens)]))

    at(most)
    tab = torch.empty(1)
    plan = plan_shared_prefix(torch.zeros(B * H + 1, dtype=torch.int32, device=gpu),
                              torch.zeros(1, dtype=torch.int32, device=gpu), B, H, G, D, P)
    assert plan.shared_pages.tolist() == [0] * (B * H)
    outs = [torch.zeros((B, H * G, D), dtype=torch.bfloat16, device=gpu) for _ in layers]
    eager = [torch.zeros_like(o) for o in outs]
    args = (ic, b, layers, positions, table, loc, plan, P)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        _step(*args, outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _step(*args, outs)
    for i, lens in enumerate([most, [700, 0, 650, 100, 641], [641, 645, 650, 0, 0], [30, 20, 33, 1, 2], [0] * 5, most]):
        at(lens)
        for o in outs + eager:
            o.fill_(9.0)
        tab = torch.full((1 << 22,), float("nan"), device=gpu)  # (what eager scratch is made of)
        torch.cuda.synchronize()
        del tab
        graph.replay()
        torch.cuda.synchronize()
        found = plan.shared_pages.view(B, H)[:, 0].tolist()
        _step(*args, eager)
        for o, e in zip(outs, eager):
            assert torch.equal(o.view(torch.int16), e.view(torch.int16)), f"replay {i}"
        assert found == plan.shared_pages.view(B, H)[:, 0].tolist()
        if i == 0:
            assert found[:3] == [shared] * 3 and found[3:] == [0, 0]
        # the last layer in 64 bits over the pools as the step left them
        q, nk, _, k, v = layers[1]
        from vortex_torch.cache import set_kv_buffer_rope
        turned = set_kv_buffer_rope(k, v, q, nk, layers[1][2], loc, P, positions, table)
        n = int(ic.dense_kv_indptr[B * H])
        want, bound = _exact(turned, k, v, ic.dense_kv_indptr[:B * H + 1], ic.dense_kv_indices[:n],
                             ic.kv_last_page_len[:B * H], D ** -0.5)
        assert bool(((outs[1].view(-1, D).double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_capture_that_torch_did_not_begin_runs_paged_attention(gpu):
    import ctypes

    table = _table([(30, [40, 3])], 16, 1, 7)
    indptr, indices, last, _ = table
    q, k, v = _inputs(table, 16, 1, 2, 128, 0, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    plan = plan_shared_prefix(t[0], t[1], 2, 1, 2, 128, 16)
    shared_prefix_decode_attention(q, k, v, *t, plan)
    whole, o = torch.zeros_like(q), torch.zeros_like(q)
    lib = _hip.load_library()
    assert lib.vtx_paged_decode_attention(q.data_ptr(), whole.data_ptr(), k.data_ptr(), v.data_ptr(), k.shape[0],
                                          *(x.data_ptr() for x in t[:2]), indices.numel(), t[2].data_ptr(), 2, 1, 2,
                                          128, 16, 128 ** -0.5, torch.cuda.current_stream().cuda_stream) == 0
    with open("/proc/self/maps") as f:
        rt = ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
    side = torch.cuda.Stream(gpu)
    torch.cuda.synchronize()
    stream, graph, run = ctypes.c_void_p(side.cuda_stream), ctypes.c_void_p(), ctypes.c_void_p()
    with torch.cuda.stream(side):
        assert rt.hipStreamBeginCapture(stream, 2) == 0  # relaxed
        try:
            shared_prefix_decode_attention(q, k, v, *t, plan, out=o)
            with pytest.raises(RuntimeError, match="needs a plan made before it"):
                plan_shared_prefix(t[0], t[1], 2, 1, 2, 128, 16)
        finally:
            assert rt.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        o.zero_()
        torch.cuda.synchronize()
        assert rt.hipGraphLaunch(run, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(o, whole)
    assert rt.hipGraphExecDestroy(run) == 0 and rt.hipGraphDestroy(graph) == 0


# ------------------------------------------------------------- refusals (CPU)
def _call(monkeypatch, **changes):
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_current_device", lambda: 0)
    i32 = dict(dtype=torch.int32)
    a = dict(q=torch.zeros((4, 2, 64), dtype=torch.bfloat16), k_cache=torch.zeros((6, 16, 64), dtype=torch.bfloat16),
             v_cache=torch.zeros((6, 16, 64), dtype=torch.bfloat16), kv_indptr=torch.zeros(5, **i32),
             kv_indices=torch.zeros(4, **i32), kv_last_page_len=torch.zeros(4, **i32),
             plan=SharedPrefixPlan(torch.zeros(4096, **i32), 2, 2, 2, 64, 16))
    a.update(changes)
    return shared_prefix_decode_attention(**a)


@pytest.mark.parametrize("changes, says", [
    (dict(q=torch.zeros((4, 2, 64))), "q must be torch.bfloat16"),
    (dict(q=torch.zeros((4, 1, 64), dtype=torch.bfloat16)), "must hold"),
    (dict(q=torch.zeros((4, 2, 128), dtype=torch.bfloat16)[..., ::2]), "q must be contiguous"),
    (dict(out=torch.zeros((4, 1, 64), dtype=torch.bfloat16)), "must hold"),
    (dict(k_cache=torch.zeros((6, 32, 64), dtype=torch.bfloat16)), "as planned"),
    (dict(k_cache=torch.zeros((6, 16, 128), dtype=torch.bfloat16)), "as planned"),
    (dict(v_cache=torch.zeros((5, 16, 64), dtype=torch.bfloat16)), "must both be"),
    (dict(v_cache=torch.zeros((6, 16, 64), dtype=torch.float16)), "v_cache must be torch.bfloat16"),
    (dict(kv_indptr=torch.zeros(4, dtype=torch.int32)), "kv_indptr needs 5"),
    (dict(kv_last_page_len=torch.zeros(3, dtype=torch.int32)), "kv_last_page_len 4"),
    (dict(kv_indices=torch.zeros(4, dtype=torch.int64)), "kv_indices must be torch.int32"),
])
def test_attention_refusals(monkeypatch, changes, says):
    with pytest.raises(RuntimeError, match=says):
        _call(monkeypatch, **changes)


@pytest.mark.parametrize("changes, says", [
    (dict(kv_indptr=torch.zeros(5, dtype=torch.int64)), "kv_indptr must be torch.int32"),
    (dict(kv_indptr=torch.zeros(4, dtype=torch.int32)), "kv_indptr needs 5"),
    (dict(group_ids=torch.zeros(1, dtype=torch.int32)), "group_ids needs 2"),
    (dict(group_ids=torch.zeros(2, dtype=torch.int64)), "group_ids must be torch.int32"),
    (dict(batch_size=-1), "must be positive"),
    (dict(num_kv_heads=0), "must be positive"),
    (dict(page_size=0), "must be positive"),
    (dict(head_dim=96), "not supported"),
    (dict(group_size=9), "not supported"),
    (dict(plan=SharedPrefixPlan(torch.zeros(64, dtype=torch.int32), 2, 2, 1, 64, 16)), "plan is for"),
])
def test_plan_refusals(monkeypatch, changes, says):
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_current_device", lambda: 0)
    a = dict(kv_indptr=torch.zeros(5, dtype=torch.int32), kv_indices=torch.zeros(4, dtype=torch.int32), batch_size=2,
             num_kv_heads=2, group_size=2, head_dim=64, page_size=16)
    a.update(changes)
    with pytest.raises(RuntimeError, match=says):
        plan_shared_prefix(**a)


def test_calls_run_on_the_tensors_device(monkeypatch):
    """With another device current, each call makes its tensors' one current and puts the other back."""
    from vortex_torch.cache import set_kv_buffer_rope

    now, seen = {"device": 1}, []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, now["device"])) or (1024 if name.endswith("_len") else 0)

    monkeypatch.setattr(_hip, "_lib", Lib())
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_current_device", lambda: now["device"])
    monkeypatch.setattr(_hip, "_stream_of", lambda index: 0)
    monkeypatch.setattr(_hip, "_scratch_lasts", lambda stream: True)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: now.update(device=d))
    i32, bf = dict(dtype=torch.int32), dict(dtype=torch.bfloat16)
    tables = torch.zeros(5, **i32), torch.zeros(4, **i32)
    plan = SharedPrefixPlan(torch.zeros(512, **i32), 2, 2, 2, 64, 16)
    assert plan_shared_prefix(*tables, 2, 2, 2, 64, 16, plan=plan) is plan
    pools = torch.zeros((2, 6, 16, 64), **bf)
    shared_prefix_decode_attention(torch.zeros((4, 2, 64), **bf), pools[0], pools[1], *tables,
                                   torch.zeros(4, **i32), plan)
    rows = torch.zeros((3, 2, 64), **bf)
    set_kv_buffer_rope(pools[0], pools[1], rows, rows.clone(), rows.clone(), torch.arange(3), 16, torch.arange(3),
                       torch.zeros((8, 64)))
    assert now["device"] == 1 and {d for _, d in seen} == {0}
    names = [n for n, _ in seen]
    for n in ("vtx_plan_shared_prefix", "vtx_shared_prefix_decode_attention", "vtx_set_kv_buffer_rope"):
        assert names.count(n) == 1


def test_attention_without_memory_for_its_scratch_raises(monkeypatch):
    """No other operator takes its place: what a call gives does not depend on the memory that is free."""
    called = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: called.append(name) or (1024 if name.endswith("_len") else 0)

    def full(*a, **k):
        raise torch.OutOfMemoryError("full")

    monkeypatch.setattr(_hip, "_lib", Lib())
    monkeypatch.setattr(_hip, "_stream_of", lambda index: 0)
    monkeypatch.setattr(_hip, "_scratch_lasts", lambda stream: True)
    out = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    monkeypatch.setattr(torch, "empty", full)
    with pytest.raises(torch.OutOfMemoryError):
        _call(monkeypatch, out=out)
    assert called == ["vtx_shared_prefix_workspace_len"]


def test_need_a_gpu():
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        plan_shared_prefix(torch.zeros(5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), 2, 2, 2, 64, 16)


def test_c_refusals():
    lib = _hip.load_library()
    p = [0x10000 * (i + 1) for i in range(10)]

    def attend(q=p[0], rows=64, B=2, H=2, G=2, D=64, P=16, ws=p[8]):
        return lib.vtx_shared_prefix_decode_attention(q, p[1], p[2], p[3], rows, p[4], p[5], 10, p[6], p[7], 1 << 20,
                                                      B, H, G, D, P, 0.1, ws, 1 << 30, None)

    for kw, says in ((dict(B=-1), b"bad sizes"), (dict(H=0), b"bad sizes"), (dict(P=0), b"bad sizes"),
                     (dict(D=96), b"not supported"), (dict(G=9), b"not supported"), (dict(q=None), b"null"),
                     (dict(ws=None), b"null"), (dict(q=p[0] + 8), b"aligned"), (dict(rows=1 << 28, P=64), b"2^32"),
                     (dict(B=1 << 25), b"too many")):
        assert attend(**kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
    assert attend(B=0) == 0

    def plan(indptr=p[0], B=2, H=2, G=2, D=64, P=16):
        return lib.vtx_plan_shared_prefix(indptr, p[1], 10, None, B, H, G, D, P, p[2], 1 << 20, None)

    for kw, says in ((dict(B=-1), b"bad sizes"), (dict(P=0), b"bad sizes"), (dict(D=80), b"not supported"),
                     (dict(G=0), b"not supported"), (dict(indptr=None), b"null"), (dict(B=1 << 25), b"too many")):
        assert plan(**kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
    assert plan(B=0) == 0


def test_plain_plan_on_a_table_written_out():
    indptr = torch.tensor([0, 3, 6, 6, 8], dtype=torch.int32)
    indices = torch.tensor([4, 7, 1, 4, 7, 2, 9, 9], dtype=torch.int32)
    assert _plain_plan(indptr, indices, 4, 1) == ([0, 0, 2, 3], [2, 2, 0, 0])
    assert _plain_plan(indptr, indices, 4, 1, [1, 2, 2, 2]) == ([0, 1, 2, 3], [0, 0, 0, 0])
    assert np.array_equal(indptr.diff().numpy(), [3, 3, 0, 2])
