"""The position-rotating cache append and shared-prefix decode attention, as
measurable cases with their plain forms.

Three kinds of pass:

``rope``    set_kv_buffer_rope: queries and new keys rotated to their
            positions, keys and values stored in the paged pools.
``plan``    plan_shared_prefix: which requests of a block table share leading
            pages, and how many.
``attend``  plan_shared_prefix once, then shared_prefix_decode_attention of
            several layers over that table, as a decode step does.

Lengths are a function of the case alone; the seed decides the block tables
and all values.
"""
from __future__ import annotations

import math
import os
import random
import sys
from types import SimpleNamespace

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _framework():
    pkg = os.path.join(os.getcwd(), "vortex_torch-dev_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from vortex_torch import cache, decode_attention

    return cache, decode_attention


# ------------------------------------------------------------------- cases
def _rope(name, tokens, q_heads, heads, dim, rotary, page=16, dtype="bf16", interleaved=False, fused=True, padding=0,
          decode=False):
    c = {"kind": "rope", "tokens": tokens, "q_heads": q_heads, "heads": heads, "dim": dim, "rotary": rotary,
         "page": page, "dtype": dtype, "interleaved": interleaved, "fused": fused, "padding": padding,
         "decode": decode}
    return dict(c, name=name) if name else c


def _plan(name, groups, per_group, prefix, suffix, heads=8, group=2, dim=128, page=16, lone=0):
    c = {"kind": "plan", "groups": groups, "per_group": per_group, "lone": lone, "prefix": prefix, "suffix": suffix,
         "heads": heads, "group": group, "dim": dim, "page": page}
    return dict(c, name=name) if name else c


def _attend(name, groups, per_group, prefix, suffix, layers, heads=8, group=2, dim=128, page=16):
    return dict(_plan(name, groups, per_group, prefix, suffix, heads, group, dim, page), kind="attend", layers=layers)


def listed():
    return [
        # one user's decode step: one token, the smallest call, latency alone
        _rope("rope_decode_1", 1, 16, 8, 128, 128, decode=True),
        # a captured decode step of 256 requests, 11 of them padding
        _rope("rope_decode_256", 256, 16, 8, 128, 128, padding=11, decode=True),
        # a chunk of prompts: neighbouring pairs, half of each row rotated, fp16, tensors of their own
        _rope("rope_prefill_8191_pairs", 8191, 32, 4, 128, 64, page=32, dtype="fp16", interleaved=True, fused=False),
        # the largest prefill chunk, out of one qkv projection
        _rope("rope_prefill_65536", 65536, 16, 8, 128, 128),
        # an ordinary server's table: two system prompts, and five requests without one
        _plan("plan_64x8k", 2, 32, 8192, 1024, lone=5),
        # many prompts, eight samples of each, some lone requests among them: the largest table
        _plan("plan_32x8x16k", 32, 8, 16384, 2048, lone=9),
        # four samples of one short prompt: the smallest call, latency and launches
        _attend("attend_4x1k", 1, 4, 1024, 64, 2),
        # 64 users behind one system prompt of 8k tokens
        _attend("attend_64x8k", 1, 64, 8192, 1024, 2),
        # 32 prompts of 4k tokens with eight samples each
        _attend("attend_32x8x4k", 32, 8, 4096, 256, 2),
        # wide rows in larger pages, one kv head group of four, odd lengths
        _attend("attend_17x5k_wide", 1, 17, 5000, 333, 2, heads=4, group=4, dim=256, page=32),
        # narrow rows, one query head each, a long shared document
        _attend("attend_48x32k_narrow", 1, 48, 32768, 512, 2, heads=8, group=1, dim=64),
        # a full server behind one long shared document: the largest call, bound by the matrix products
        _attend("attend_256x16k", 1, 256, 16384, 512, 2, heads=8, group=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "plan", "attend", "attend", "attend"])
    heads = rng.choice([1, 2, 4, 8, 8])
    page = rng.choice([16, 16, 32, 64])
    if kind == "rope":
        dim = rng.choice([64, 80, 128, 128, 256])
        group = rng.choice([1, 2, 4, 8])
        rotary = rng.choice([dim, dim, dim // 2])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        row = (heads * group + 2 * heads) * dim * (4 if dtype == "fp32" else 2)
        tokens = _log(rng, 1, max(2, min(65536, 65536 * 8192 // row)))
        decode = tokens <= 512 and rng.random() < 0.7
        return _rope(None, tokens, heads * group, heads, dim, rotary, page=page, dtype=dtype,
                     interleaved=rng.random() < 0.3, fused=rng.random() < 0.6,
                     padding=rng.randint(0, tokens // 4) if decode else 0, decode=decode)
    groups = _log(rng, 1, 64)
    per_group = _log(rng, 1 if groups > 1 else 2, max(2, 256 // groups))
    suffix = _log(rng, 1, 1024)
    prefix = _log(rng, 64, 32768)
    if kind == "plan":
        prefix = max(1, min(prefix, 256 * 10240 // (groups * per_group)))
        return _plan(None, groups, per_group, prefix, suffix, heads=heads, group=rng.choice([1, 2, 4, 8]), page=page,
                     lone=rng.randint(4, 16))
    group = rng.choice([1, 2, 2, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    # no dearer than the largest listed case, in products and in bytes
    most = (1 << 30) // (10 * heads * dim * groups)  # tokens of a group
    each = 256 * 16384 * 8 * 8 * 128 // (groups * per_group * group * heads * dim) - suffix  # tokens seen by a request
    suffix = max(1, min(suffix, most // (2 * per_group)))
    prefix = max(1, min(prefix, most // 2, each))
    return _attend(None, groups, per_group, prefix, suffix, 2, heads=heads, group=group, dim=dim, page=page)


# ------------------------------------------------------------------ inputs
def _gen(seed, *what):
    return torch.Generator(device="cuda").manual_seed(random.Random(f"{seed} {what}").randrange(1 << 62))


def _randn(shape, gen, dtype=torch.bfloat16, std=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    return t.mul_(std) if std != 1.0 else t


def _prepare_rope(case, seed):
    """A step's projections, the pools and tables that a runtime holds."""
    n, Hq, H, D, P = case["tokens"], case["q_heads"], case["heads"], case["dim"], case["page"]
    dtype = _DTYPES[case["dtype"]]
    if case["fused"]:  # slices of one projection's rows
        qkv = _randn((n, (Hq + 2 * H) * D), _gen(seed, "qkv"), dtype)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, H * D, H * D], dim=1))
    else:
        q, k, v = (_randn((n, h, D), _gen(seed, w), dtype) for w, h in (("q", Hq), ("k", H), ("v", H)))
    pages = (n + P - 1) // P + max(8, n // (8 * P))
    perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
    tok = torch.arange(n, device="cuda")
    last = 131072
    if case["decode"]:  # every request at a length of its own, its newest token in a page of its own
        pages = n + 8
        perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
        positions = torch.randint(0, last, (n,), generator=_gen(seed, "positions"), device="cuda")
        loc = perm[:n] * P + positions % P
    else:  # chunks of consecutive tokens, the first somewhere in its request
        positions = (tok + random.Random(f"start {seed}").randrange(last)) % last
        loc = perm[tok // P] * P + tok % P
    real = n - case["padding"]
    loc[real:] = -1
    positions[real:] = 0
    half = case["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * freq
    table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
    kc, vc = (_randn((pages * H, P, D), _gen(seed, w), dtype) for w in ("k_cache", "v_cache"))
    return SimpleNamespace(case=case, q=q, k=k, v=v, loc=loc, positions=positions, table=table, k_cache=kc, v_cache=vc,
                           real=real)


def _lengths(case):
    """Every request's (group, pages shared with it, own tokens); a lone
    request has a group to itself and shares nothing."""
    r = random.Random(f"{case['groups']} {case['per_group']} {case['prefix']} {case['suffix']}")
    shared = [case["prefix"]] + [r.randint(max(1, case["prefix"] // 2), case["prefix"])
                                 for _ in range(case["groups"] - 1)]
    got = [(g, max(1, shared[g] // case["page"]), r.randint(1, case["suffix"]))
           for g in range(case["groups"]) for _ in range(case["per_group"])]
    got[0] = got[0][:2] + (case["suffix"],)
    return got + [(case["groups"] + i, 0, r.randint(1, case["suffix"])) for i in range(case["lone"])]


def _table(case, seed):
    """The batch's dense block table, pages drawn from one shuffled pool; the
    seed decides the order of the groups."""
    P, H = case["page"], case["heads"]
    r = random.Random(f"order {seed}")
    order = list(range(case["groups"] + case["lone"]))
    r.shuffle(order)
    batch = sorted(_lengths(case), key=lambda x: order[x[0]])
    shared = {g: pages for g, pages, _ in batch}
    own_pages = [(t + P - 1) // P for _, _, t in batch]
    used = sum(shared.values()) + sum(own_pages)
    pool = used + max(64, used // 16)
    perm = torch.randperm(pool, generator=_gen(seed, "pages"), device="cuda").to(torch.int32)
    *parts, _ = perm.split([*shared.values(), *own_pages, pool - used])
    prefix = dict(zip(shared, parts))
    heads = torch.arange(H, device="cuda", dtype=torch.int32)[:, None]
    rows = [(torch.cat([prefix[g], tail])[None, :] * H + heads).reshape(-1)
            for (g, _, _), tail in zip(batch, parts[len(shared):])]
    count = [p + o for (_, p, _), o in zip(batch, own_pages)]
    i32 = dict(dtype=torch.int32, device="cuda")
    ends = torch.tensor(count, **i32).repeat_interleave(H).cumsum(0, dtype=torch.int32)
    return SimpleNamespace(
        case=case, pool=pool, batch=len(batch), indices=torch.cat(rows), indptr=torch.cat([torch.zeros(1, **i32), ends]),
        last=torch.tensor([(t - 1) % P + 1 for _, _, t in batch], **i32).repeat_interleave(H), longest=max(count),
        longest_prefix=max(shared.values()), longest_suffix=max(own_pages),
        shared=torch.tensor(list(shared.values()), device="cuda"))


def _prepare_attend(case, seed):
    s = _table(case, seed)
    P, H, G, D = case["page"], case["heads"], case["group"], case["dim"]
    rows = s.pool * H
    s.layers = [SimpleNamespace(q=_randn((s.batch * H, G, D), _gen(seed, i, "q"), std=1.5),
                                k=_randn((rows, P, D), _gen(seed, i, "k")),
                                v=_randn((rows, P, D), _gen(seed, i, "v"))) for i in range(case["layers"])]
    return s


def prepare(case, seed):
    return {"rope": _prepare_rope, "plan": _table, "attend": _prepare_attend}[case["kind"]](case, seed)


# ------------------------------------------------------------------ passes
def _turn(x, s, real=None):
    """x [n, heads, D] rotated to its tokens' positions, in fp32, rounded once."""
    R = s.case["rotary"]
    x = x.float()
    cs = s.table[s.positions][:, None, :]
    cos, sin = cs[..., :R // 2], cs[..., R // 2:]
    if s.case["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([out, x[..., R:]], dim=-1).to(s.q.dtype)


def _plain_rope(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    loc = s.loc[:s.real]
    for_k, for_v = s.k_cache.view(-1, H, P, D), s.v_cache.view(-1, H, P, D)
    for_k[loc // P, :, loc % P] = _turn(s.k, s)[:s.real]
    for_v[loc // P, :, loc % P] = s.v[:s.real]
    return {"q": _turn(s.q, s), "k_cache": s.k_cache, "v_cache": s.v_cache}


def _padded(s, first, count, longest):
    """Entries [first, first + count) of every segment, [B, H, longest], -1 past its end."""
    at = torch.arange(longest, device="cuda")
    idx = first[:, None] + at
    got = s.indices[idx.clamp(max=s.indices.numel() - 1)]
    return torch.where(at < count[:, None], got, -1).view(s.batch, s.case["heads"], longest)


def _plain_plan(s):
    H, B = s.case["heads"], s.batch
    start, pages = s.indptr[:-1].long(), s.indptr.diff().long()
    rows = _padded(s, start, pages, s.longest)
    same = rows[1:, :, 0] == rows[:-1, :, 0]  # with the request before
    lone = torch.zeros((1, H), dtype=torch.bool, device="cuda")
    same = torch.cat([lone, same])
    common = ((rows[1:] == rows[:-1]) & (rows[1:] >= 0)).long().cumprod(-1).sum(-1)
    limit = pages.view(B, H) - 1
    common = torch.cat([limit[:1], torch.where(same[1:], common, limit[1:])])  # (a run's first: its own pages)
    b = torch.arange(B, device="cuda")[:, None].expand(B, H)
    leader = torch.where(same, 0, b).cummax(0).values
    shared = torch.full((B, H), 1 << 30, device="cuda").scatter_reduce(0, leader, torch.minimum(common, limit), "amin")
    alone = torch.zeros((B, H), device="cuda", dtype=torch.long).scatter_add(0, leader, torch.ones_like(leader)) == 1
    shared = torch.where(alone, 0, shared).gather(0, leader)
    return {"leaders": leader.to(torch.int32).flatten(), "shared_pages": shared.to(torch.int32).flatten()}


def _plain_attend(s):
    """The shared pages once for all requests of a group, every request's own
    pages, and one softmax over both."""
    c = s.case
    P, H, G, D, n, NG, B = c["page"], c["heads"], c["group"], c["dim"], c["per_group"], c["groups"], s.batch
    start, pages = s.indptr[:-1].long(), s.indptr.diff().long()
    shared = s.shared.repeat_interleave(n * H)
    prefix = _padded(s, start, shared, s.longest_prefix).view(NG, n, H, -1)[:, 0]
    suffix = _padded(s, start + shared, pages - shared, s.longest_suffix)
    tokens = (pages - shared - 1) * P + s.last
    seen_p = (prefix >= 0).repeat_interleave(P, -1)[:, :, None, :]
    seen_s = (torch.arange(s.longest_suffix * P, device="cuda") < tokens[:, None]).view(B, H, 1, -1)
    wide = lambda pool, rows: pool[rows.clamp(min=0)].flatten(2, 3).float()  # noqa: E731

    def layer(x):
        q = x.q.float().view(NG, n, H, G, D) / math.sqrt(D)
        qg = q.transpose(1, 2).reshape(NG, H, n * G, D)
        qs = q.reshape(B, H, G, D)
        sp = (qg @ wide(x.k, prefix).transpose(-1, -2).contiguous()).masked_fill(~seen_p, -math.inf)
        ss = (qs @ wide(x.k, suffix).transpose(-1, -2).contiguous()).masked_fill(~seen_s, -math.inf)
        by_row = lambda t: t.reshape(NG, H, n, G, -1).transpose(1, 2).reshape(B, H, G, -1)  # noqa: E731
        to_group = lambda t: t.reshape(NG, n, H, G, 1).transpose(1, 2).reshape(NG, H, n * G, 1)  # noqa: E731
        top = torch.maximum(by_row(sp.amax(-1)), ss.amax(-1, keepdim=True))
        sp = sp.sub_(to_group(top)).exp_()
        ss = ss.sub_(top).exp_()
        weight = by_row(sp.sum(-1)) + ss.sum(-1, keepdim=True)
        o = by_row(sp @ wide(x.v, prefix)) + ss @ (wide(x.v, suffix) * seen_s.transpose(-1, -2))
        return (o / weight).to(x.q.dtype).reshape(x.q.shape)

    return [layer(x) for x in s.layers]


def run(state):
    s, c = state, state.case
    if not own:
        return {"rope": _plain_rope, "plan": _plain_plan, "attend": _plain_attend}[c["kind"]](s)
    cache, attention = _framework()
    if c["kind"] == "rope":
        q = cache.set_kv_buffer_rope(s.k_cache, s.v_cache, s.q, s.k, s.v, s.loc, c["page"], s.positions, s.table,
                                     interleaved=c["interleaved"])
        return {"q": q, "k_cache": s.k_cache, "v_cache": s.v_cache}
    plan = attention.plan_shared_prefix(s.indptr, s.indices, s.batch, c["heads"], c["group"], c["dim"], c["page"])
    if c["kind"] == "plan":
        return {"leaders": plan.leaders, "shared_pages": plan.shared_pages}
    return [attention.shared_prefix_decode_attention(x.q, x.k, x.v, s.indptr, s.indices, s.last, plan)
            for x in s.layers]


def work(case):
    if case["kind"] == "rope":
        n, R, D = case["tokens"], case["rotary"], case["dim"]
        size = 4 if case["dtype"] == "fp32" else 2
        heads = case["q_heads"] + 2 * case["heads"]
        stored = n * case["q_heads"] + (n - case["padding"]) * 2 * case["heads"]
        return {"bytes": (n * heads + stored) * D * size + n * (16 + 4 * R),
                "flops": 3 * R * n * (case["q_heads"] + case["heads"])}
    P, H, batch = case["page"], case["heads"], _lengths(case)
    entries = H * sum(p + (t + P - 1) // P for _, p, t in batch)
    if case["kind"] == "plan":
        return {"bytes": 4 * entries + 12 * H * len(batch), "flops": 0}
    G, D = case["group"], case["dim"]
    read = P * sum({g: p for g, p, _ in batch}.values()) + sum(t for _, _, t in batch)  # distinct tokens
    seen = sum(p * P + t for _, p, t in batch)
    per_layer = 4 * H * D * read + 4 * H * G * D * len(batch)
    return {"bytes": case["layers"] * per_layer + 4 * entries + 4 * H * len(batch),
            "flops": case["layers"] * 4 * D * G * H * seen}


# ---------------------------------------------------------- in 64 bits
def _exact_rope(s):
    """The rotation as a product of complex numbers; stored token by head."""
    c = s.case
    R, H, P, D = c["rotary"], c["heads"], c["page"], c["dim"]
    row = s.table.double()[s.positions]
    unit = torch.complex(row[:, :R // 2], row[:, R // 2:])[:, None]

    def turned(x):
        y = x.double().clone()
        pairs = y[..., :R].unflatten(-1, (R // 2, 2) if c["interleaved"] else (2, R // 2))
        if not c["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
        y[..., :R] = (z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return y

    keep = s.loc >= 0
    row0 = (s.loc[keep] // P) * (P * H) + s.loc[keep] % P
    at = row0[:, None] + torch.arange(H, device="cuda") * P
    kc, vc = (t.double().view(-1, D) for t in (s.k_cache, s.v_cache))
    kc[at.flatten()] = turned(s.k)[keep].flatten(0, 1)
    vc[at.flatten()] = s.v.double()[keep].flatten(0, 1)
    return {"q": turned(s.q), "k_cache": kc.view(s.k_cache.shape), "v_cache": vc.view(s.v_cache.shape)}


def _exact_attend(s):
    """Full attention of every segment over all its tokens, one by one."""
    c = s.case
    P, G, D, H = c["page"], c["group"], c["dim"], c["heads"]
    ptr, last = s.indptr.tolist(), s.last.tolist()

    def segment(x, i):
        rows = s.indices[ptr[i]:ptr[i + 1]].long()
        n = (rows.numel() - 1) * P + last[i]
        k, v = (t[rows].reshape(-1, D)[:n].double() for t in (x.k, x.v))
        return torch.softmax(x.q[i].double() @ k.t().contiguous() * D ** -0.5, dim=-1) @ v

    return [torch.stack([segment(x, i) for i in range(s.batch * H)]) for x in s.layers]


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_rope(s) if case["kind"] == "rope" else _exact_attend(s)
