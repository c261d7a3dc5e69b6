"""The 8-bit paged cache, as measurable cases with their plain forms: pools of
e4m3 or int8 codes, and one power of two per token, kv head and K or V.

Four kinds of pass:

``append``  set_kv_buffer_quant: new keys and values quantised into the pools.
``read``    read_kv_buffer_quant: the values at given slots.
``pages``   the page-finish reductions of keys held in 8 bits.
``attend``  decode attention of one new token per request over the pools, by a
            dense table or one of selected pages; with capped scores, a window
            or a bias that grows with the distance.

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
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# a format's largest code as m * 2^x, m in [0.5, 1): 448 and 127
_TOP = {"e4m3": (0.875, 9), "int8": (0.9921875, 7)}


def _framework():
    pkg = os.path.join(os.getcwd(), "vortex_torch-dev_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from vortex_torch import abs as vabs
    from vortex_torch import cache, decode_attention, utils

    return cache, decode_attention, vabs, utils


# ------------------------------------------------------------------- cases
def _append(name, tokens, heads, dim, page=16, dtype="bf16", codes="e4m3", fused=True, padding=0, decode=False):
    c = {"kind": "append", "tokens": tokens, "heads": heads, "dim": dim, "page": page, "dtype": dtype, "codes": codes,
         "fused": fused, "padding": padding, "decode": decode}
    return dict(c, name=name) if name else c


def _read(name, tokens, heads, dim, page=16, dtype="bf16", codes="e4m3"):
    c = {"kind": "read", "tokens": tokens, "heads": heads, "dim": dim, "page": page, "dtype": dtype, "codes": codes}
    return dict(c, name=name) if name else c


def _pages(name, tokens, heads, dim, page=16, codes="e4m3", envelope=False, decode=False):
    c = {"kind": "pages", "tokens": tokens, "heads": heads, "dim": dim, "page": page, "codes": codes,
         "envelope": envelope, "decode": decode}
    return dict(c, name=name) if name else c


def _attend(name, batch, longest, heads=8, group=2, dim=128, page=16, dtype="bf16", codes="e4m3", sparse=False, cap=0.0,
            window=0, slopes=False):
    c = {"kind": "attend", "batch": batch, "longest": longest, "heads": heads, "group": group, "dim": dim, "page": page,
         "dtype": dtype, "codes": codes, "sparse": sparse, "cap": cap, "window": window, "slopes": slopes}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's decode step: one token, the smallest call, latency alone
        _append("append_decode_1", 1, 8, 128, decode=True),
        # a captured decode step of 256 requests, 11 of them padding
        _append("append_decode_256", 256, 8, 128, codes="int8", padding=11, decode=True),
        # a chunk of prompts: fp16 tensors of their own, rows of 80 columns, larger pages
        _append("append_prefill_8191", 8191, 4, 80, page=32, dtype="fp16", codes="int8", fused=False),
        # the largest prefill chunk, out of one qkv projection
        _append("append_prefill_65536", 65536, 8, 128),
        # one request's prefix, read back for the next chunk of its prompt
        _read("read_5000", 5000, 4, 128, dtype="fp16", codes="int8"),
        # the prefixes of a whole batch
        _read("read_131072", 131072, 8, 128),
        # a decode step of 64 requests, of whose pages a few are full now
        _pages("pages_decode_64", 64, 8, 128, decode=True),
        # the pages of a burst of prompts, their keys' maxima and minima
        _pages("pages_burst_262144", 262144, 8, 128, codes="int8", envelope=True),
        # one user's decode step behind 4k tokens: latency alone
        _attend("attend_1x4k", 1, 4096),
        # an ordinary sparse step: 64 requests, 32 selected pages each
        _attend("attend_sparse_64", 64, 512, codes="int8", sparse=True),
        # capped scores and a window, wide rows in larger pages, ragged lengths
        _attend("attend_48x8k_capped", 48, 8192, heads=4, group=4, dim=256, page=32, codes="int8", cap=50.0,
                window=4096),
        # the largest: long documents, eight query heads each
        _attend("attend_32x32k", 32, 32768, group=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "pages", "attend", "attend", "attend"])
    heads = rng.choice([1, 2, 4, 8, 8])
    page = rng.choice([16, 16, 32, 64])
    codes = rng.choice(["e4m3", "int8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    if kind == "attend":
        dim = rng.choice([64, 128, 128, 256])
        group = rng.choice([1, 2, 4, 8, 16])
        batch = _log(rng, 1, 256)
        sparse = rng.random() < 0.3
        # no dearer than the largest listed case, in bytes and in products
        most = 32 * 32768 * 8 * 128 // (batch * heads * dim)
        most = min(most, 8 * most // group)
        longest = max(1, min(_log(rng, 1, 32768), most))
        if sparse:
            longest = max(page, min(longest, 64 * page) // page * page)
        return _attend(None, batch, longest, heads=heads, group=group, dim=dim, page=page,
                       dtype=rng.choice(["bf16", "bf16", "fp16"]), codes=codes, sparse=sparse,
                       cap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                       window=0 if sparse or rng.random() < 0.7 else _log(rng, 16, 8192),
                       slopes=not sparse and rng.random() < 0.2)
    dim = rng.choice([64, 80, 128, 128, 256])
    if kind == "append":
        tokens = _log(rng, 1, max(2, min(65536, 65536 * 8 * 128 * 2 // (heads * dim * size))))
        decode = tokens <= 512 and rng.random() < 0.7
        return _append(None, tokens, heads, dim, page=page, dtype=dtype, codes=codes, fused=rng.random() < 0.6,
                       padding=rng.randint(0, tokens // 4) if decode else 0, decode=decode)
    if kind == "read":
        tokens = _log(rng, 1, max(2, min(131072, 131072 * 8 * 128 * 2 // (heads * dim * size))))
        return _read(None, tokens, heads, dim, page=page, dtype=dtype, codes=codes)
    decode = rng.random() < 0.4
    dim = rng.choice([64, 128, 128, 256])
    tokens = _log(rng, 1, 512 if decode else max(2, min(262144, 262144 * 8 * 128 // (heads * dim))))
    return _pages(None, tokens, heads, dim, page=page, codes=codes, envelope=rng.random() < 0.4, decode=decode)


# ------------------------------------------------------------------ inputs
def _gen(seed, *what):
    return torch.Generator(device="cuda").manual_seed(random.Random(f"{seed} {what}").randrange(1 << 62))


def _randn(shape, gen, dtype=torch.bfloat16, std=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    return t.mul_(std) if std != 1.0 else t


def _quantise(x, codes):
    """Rows x [..., D] as codes and exponent bytes, in their plain form: the
    least power of two by which the row's largest value fits the codes."""
    x = x.float()
    top, bits = _TOP[codes]
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, e - bits + (m > top).int(), -126).clamp(min=-126)
    y = torch.ldexp(x, -e[..., None])
    return (y.round().to(torch.int8) if codes == "int8" else y.to(torch.float8_e4m3fn)), (e + 127).to(torch.uint8)


def _factor(b):
    """What an exponent byte stands for."""
    return torch.ldexp(torch.ones_like(b, dtype=torch.float32), b.int() - 127)


def _bytes(t):
    return t.view(torch.uint8)


def _pools(rows, page, dim, codes, seed):
    """Pools that hold older tokens: keys whose columns have sizes of their
    own, values; made some rows at a time."""
    kc, vc = (torch.empty((rows, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = torch.empty((rows, page, 2), dtype=torch.uint8, device="cuda")
    size = _randn((dim,), _gen(seed, "columns"), torch.float32).mul(0.3).exp().bfloat16()
    step = max(1, (1 << 26) // (page * dim))
    for i, (pool, what) in enumerate(((kc, "k"), (vc, "v"))):
        gen = _gen(seed, what, "pool")
        for r in range(0, rows, step):
            x = _randn((min(step, rows - r), page, dim), gen)
            c, b = _quantise(x * size if what == "k" else x, codes)
            pool[r:r + step], scales[r:r + step, :, i] = _bytes(c), b
    return kc.view(_CODES[codes]), vc.view(_CODES[codes]), scales


def _slots(n, page, pages, start, seed):
    """Slots of chunks of consecutive tokens, the first `start` slots into its page."""
    perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
    tok = torch.arange(start, start + n, device="cuda")
    return perm[tok // page] * page + tok % page


def _prepare_append(case, seed):
    """A step's keys and values, the pools that a runtime holds."""
    n, H, D, P = case["tokens"], case["heads"], case["dim"], case["page"]
    dtype = _DTYPES[case["dtype"]]
    if case["fused"]:  # slices of one projection's rows, twice as many query heads before them
        qkv = _randn((n, 4 * H * D), _gen(seed, "qkv"), dtype)
        _, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([2 * H * D, H * D, H * D], dim=1))
    else:
        k, v = (_randn((n, H, D), _gen(seed, w), dtype) for w in ("k", "v"))
    if case["decode"]:  # every request's newest token in a page of its own
        pages = n + 8
        perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
        loc = perm[:n] * P + torch.randint(0, P, (n,), generator=_gen(seed, "slots"), device="cuda")
    else:
        pages = (n + 2 * P - 2) // P + max(8, n // (8 * P))
        loc = _slots(n, P, pages, random.Random(f"start {seed}").randrange(P), seed)
    real = n - case["padding"]
    loc[real:] = -1
    kc, vc, scales = _pools(pages * H, P, D, case["codes"], seed)
    return SimpleNamespace(case=case, k=k, v=v, loc=loc, k_cache=kc, v_cache=vc, scales=scales, real=real)


def _prepare_read(case, seed):
    n, H, D, P = case["tokens"], case["heads"], case["dim"], case["page"]
    pages = (n + P - 1) // P + max(8, n // (8 * P))
    kc, vc, scales = _pools(pages * H, P, D, case["codes"], seed)
    return SimpleNamespace(case=case, loc=_slots(n, P, pages, 0, seed), k_cache=kc, v_cache=vc, scales=scales)


def _prepare_pages(case, seed):
    n, H, D, P = case["tokens"], case["heads"], case["dim"], case["page"]
    if case["decode"]:
        pages = n + 64
        perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")
        r = random.Random(f"slots {seed}")
        slots = [P - 1 if i % P == 0 else r.randrange(P) for i in range(n)]
        loc = perm[:n] * P + torch.tensor(slots, device="cuda")
    else:
        pages = (n + P - 1) // P + max(8, n // (8 * P))
        loc = _slots(n, P, pages, 0, seed)
    kc, _, scales = _pools(pages * H, P, D, case["codes"], seed)
    out = [_randn((pages * H, 1, D), _gen(seed, "out", i)) for i in range(2 if case["envelope"] else 1)]
    return SimpleNamespace(case=case, loc=loc, k_cache=kc, scales=scales, out=out, pages=pages, op=None)


def _lengths(case):
    """Every request's tokens: the longest, and others down to an eighth of
    it; selected pages are as many for all, the last one partly filled."""
    r = random.Random(f"{case['batch']} {case['longest']} {case['page']}")
    n = case["longest"]
    if case["sparse"]:
        return [n - r.randrange(case["page"]) for _ in range(case["batch"])]
    return [n] + [r.randint(max(1, n // 8), n) for _ in range(case["batch"] - 1)]


def _prepare_attend(case, seed):
    """A batch's block table, pages drawn from one shuffled pool (selected
    ones: other pages in every head), the pools and the new token's queries."""
    B, H, G, D, P = case["batch"], case["heads"], case["group"], case["dim"], case["page"]
    tokens = _lengths(case)
    count = [(t + P - 1) // P for t in tokens]
    used = sum(count)
    pages = used + max(64, used // 16)
    heads = torch.arange(H, device="cuda", dtype=torch.int32)
    if case["sparse"]:
        perm = torch.stack([torch.randperm(pages, generator=_gen(seed, "pages", h), device="cuda")[:used]
                            for h in range(H)]).to(torch.int32)
    else:
        perm = torch.randperm(pages, generator=_gen(seed, "pages"), device="cuda")[:used].to(torch.int32).expand(H, -1)
    indices = torch.cat([p.reshape(-1) for p in (perm * H + heads[:, None]).split(count, dim=1)])
    i32 = dict(dtype=torch.int32, device="cuda")
    ends = torch.tensor(count, **i32).repeat_interleave(H).cumsum(0, dtype=torch.int32)
    kc, vc, scales = _pools(pages * H, P, D, case["codes"], seed)
    slopes = None
    if case["slopes"]:  # 2^(-8 i / heads)
        slopes = torch.exp2(-8 * torch.arange(1, H * G + 1, device="cuda", dtype=torch.float32) / (H * G))
    return SimpleNamespace(
        case=case, q=_randn((B, H * G, D), _gen(seed, "q"), _DTYPES[case["dtype"]], std=1.5), k_cache=kc, v_cache=vc,
        scales=scales, indices=indices, indptr=torch.cat([torch.zeros(1, **i32), ends]),
        last=torch.tensor([(t - 1) % P + 1 for t in tokens], **i32).repeat_interleave(H), longest=max(count),
        slopes=slopes)


def prepare(case, seed):
    return {"append": _prepare_append, "read": _prepare_read, "pages": _prepare_pages,
            "attend": _prepare_attend}[case["kind"]](case, seed)


# ------------------------------------------------------------------ passes
def _plain_append(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    loc = s.loc[:s.real]
    scales = s.scales.view(-1, H, P, 2)
    for i, (pool, x) in enumerate(((s.k_cache, s.k), (s.v_cache, s.v))):
        c, b = _quantise(x[:s.real], s.case["codes"])
        _bytes(pool).view(-1, H, P, D)[loc // P, :, loc % P] = _bytes(c)
        scales[loc // P, :, loc % P, i] = b
    return _held(s)


def _held(s):
    """The pools' codes and factors, as the numbers that they stand for."""
    return {"k_cache": s.k_cache, "v_cache": s.v_cache, "scales": s.scales.view(torch.float8_e8m0fnu)}


def _plain_read(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    f = _factor(s.scales.view(-1, H, P, 2)[s.loc // P, :, s.loc % P])
    out = []
    for i, pool in enumerate((s.k_cache, s.v_cache)):
        c = _bytes(pool).view(-1, H, P, D)[s.loc // P, :, s.loc % P].view(pool.dtype)
        out.append((c.float() * f[..., i, None]).to(_DTYPES[s.case["dtype"]]))
    return out


def _plain_pages(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    full = s.loc[(s.loc + 1) % P == 0] // P
    c = _bytes(s.k_cache).view(-1, H, P, D)[full].view(s.k_cache.dtype)
    x = c.float() * _factor(s.scales.view(-1, H, P, 2)[full][..., 0])[..., None]
    got = [x.amax(2), x.amin(2)] if s.case["envelope"] else [x.mean(2)]
    for o, y in zip(s.out, got):
        o.view(-1, H, D)[full] = y.to(o.dtype)
    return s.out


def _plain_attend(s):
    c = s.case
    B, H, G, D, P, T = c["batch"], c["heads"], c["group"], c["dim"], c["page"], s.longest * c["page"]
    start, count = s.indptr[:-1].long(), s.indptr.diff().long()
    at = torch.arange(s.longest, device="cuda")
    rows = s.indices[(start[:, None] + at).clamp(max=s.indices.numel() - 1)].long()
    rows = torch.where(at < count[:, None], rows, 0)
    f = _factor(s.scales[rows].view(B * H, T, 2))
    k = _bytes(s.k_cache)[rows].view(s.k_cache.dtype).view(B * H, T, D).float()
    x = k @ s.q.float().view(B * H, G, D).transpose(1, 2).contiguous()
    del k
    x = x * (f[..., :1] / math.sqrt(D))
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    t = torch.arange(T, device="cuda")
    tokens = ((count - 1) * P + s.last)[:, None]
    if s.slopes is not None:
        far = (tokens - 1 - t).float()[..., None]
        x = x - far * s.slopes.view(1, H, 1, G).expand(B, H, 1, G).reshape(B * H, 1, G)
    seen = (t < tokens) & (t >= tokens - c["window"]) if c["window"] else t < tokens
    x = x.masked_fill(~seen[..., None], -math.inf)
    p = (x - x.amax(1, keepdim=True)).exp_()
    total = p.sum(1)[..., None]
    p = torch.where(seen[..., None], p * f[..., 1:], 0).transpose(1, 2).contiguous()
    v = _bytes(s.v_cache)[rows].view(s.v_cache.dtype).view(B * H, T, D).float()
    return ((p @ v) / total).to(s.q.dtype).view(s.q.shape)


def _own_pages(s):
    cache, _, vabs, utils = _framework()
    c = s.case
    if s.op is None:  # as a program that keeps its operator has it
        tag = lambda t: vabs.as_vtensor(t, vabs.FORMAT.PAGED)  # noqa: E731
        ctx = cache.Context()
        ctx.page_size, ctx.head_num, ctx.head_dim, ctx.total_num_pages = c["page"], c["heads"], c["dim"], s.pages
        ctx.max_new_tokens_per_batch = c["tokens"]
        ctx.profile()
        x, outs = cache.quantized_pool(s.k_cache, s.scales), [tag(o) for o in s.out]
        op = cache.MultiReduce([utils.ReduceType.Max, utils.ReduceType.Min]) if c["envelope"] else cache.Mean()
        out = outs if c["envelope"] else outs[0]
        op(x, out, loc=s.loc, ctx=ctx)
        ctx.execute()
        s.op = lambda: op(x, out, loc=s.loc, ctx=ctx)
    s.op()
    return s.out


def run(state):
    s, c = state, state.case
    if not own:
        return {"append": _plain_append, "read": _plain_read, "pages": _plain_pages,
                "attend": _plain_attend}[c["kind"]](s)
    if c["kind"] == "pages":
        return _own_pages(s)
    cache, attention, _, _ = _framework()
    if c["kind"] == "append":
        cache.set_kv_buffer_quant(s.k_cache, s.v_cache, s.scales, s.k, s.v, s.loc, c["page"])
        return _held(s)
    if c["kind"] == "read":
        return list(cache.read_kv_buffer_quant(s.k_cache, s.v_cache, s.scales, s.loc, c["page"], c["heads"],
                                               dtype=_DTYPES[c["dtype"]]))
    return attention.quant_paged_decode_attention(
        s.q, s.k_cache, s.v_cache, s.scales, s.indptr, s.indices, s.last, c["batch"], c["heads"],
        logits_soft_cap=c["cap"], window=c["window"], slopes=s.slopes)


def work(case):
    H, D, P = case["heads"], case["dim"], case["page"]
    if case["kind"] == "attend":
        G, size = case["group"], 2
        tokens = sum(min(t, case["window"] or t) for t in _lengths(case))
        entries = H * sum((min(t, case["window"] or t) + P - 1) // P for t in _lengths(case))
        return {"bytes": 2 * H * (D + 1) * tokens + 4 * entries + case["batch"] * H * (2 * G * D * size + 8),
                "flops": 4 * H * G * D * tokens}
    n, size = case["tokens"], 4 if case.get("dtype") == "fp32" else 2
    if case["kind"] == "append":
        stored = n - case["padding"]
        return {"bytes": stored * 2 * H * (D * size + D + 1) + 8 * n, "flops": 3 * stored * 2 * H * D}
    if case["kind"] == "read":
        return {"bytes": n * 2 * H * (D * size + D + 1) + 8 * n, "flops": n * 2 * H * D}
    full = (n + P - 1) // P if case["decode"] else n // P
    outs = 2 if case["envelope"] else 1
    return {"bytes": full * H * (P * (D + 1) + outs * 2 * D) + 8 * n, "flops": full * H * P * D * (1 + outs)}


# ---------------------------------------------------------- in 64 bits
def _stored(x, codes):
    """(codes, factor) of rows x by steps through the powers of two, in 64 bits."""
    x = x.double()
    most, top = (127.0 if codes == "int8" else 448.0), x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)) - math.log2(most)).clamp(-127, 127) - 1
    for _ in range(3):
        e = torch.where(top > most * torch.exp2(e), e + 1, e)
    e = e.clamp(min=-126)
    y = x / torch.exp2(e)
    if codes == "int8":
        return torch.round(y), torch.exp2(e)
    # steps of e4m3: 2^-3 of a value's power of two, and no finer than 2^-9
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, torch.exp2(e)


def _values(pool, scales, i):
    return pool.to(torch.float64) * torch.exp2(scales[..., i].double() - 127)[..., None]


def _exact_append(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    keep = s.loc >= 0
    at = ((s.loc[keep] // P) * (P * H) + s.loc[keep] % P)[:, None] + torch.arange(H, device="cuda") * P
    scales = torch.exp2(s.scales.double() - 127).view(-1, 2)
    pools = []
    for i, (pool, x) in enumerate(((s.k_cache, s.k), (s.v_cache, s.v))):
        c, f = _stored(x[keep], s.case["codes"])
        pools.append(pool.to(torch.float64).view(-1, D))
        pools[i][at.flatten()] = c.flatten(0, 1)
        scales[at.flatten(), i] = f.flatten()
    whole = s.case["codes"] == "int8"  # (whole numbers)
    k, v = (None if whole else p.view(s.k_cache.shape) for p in pools)
    return {"k_cache": k, "v_cache": v, "scales": scales.view(s.scales.shape)}


def _exact_read(s):
    P, H, D = s.case["page"], s.case["heads"], s.case["dim"]
    at = ((s.loc // P) * (P * H) + s.loc % P)[:, None] + torch.arange(H, device="cuda") * P
    sc = s.scales.view(-1, 2)[at]
    return [_values(_bytes(p).view(-1, D)[at].view(p.dtype), sc, i) for i, p in enumerate((s.k_cache, s.v_cache))]


def _exact_pages(s):
    P, H = s.case["page"], s.case["heads"]
    out = [o.double() for o in s.out]
    full = torch.unique(s.loc[s.loc % P == P - 1] // P)
    for part in full.split(4096):
        rows = (part[:, None] * H + torch.arange(H, device="cuda")).flatten()
        x = _values(_bytes(s.k_cache)[rows].view(s.k_cache.dtype), s.scales[rows], 0)
        got = [x.max(1).values, x.min(1).values] if s.case["envelope"] else [x.sum(1) / P]
        for o, y in zip(out, got):
            o[rows, 0] = y
    return out


def _exact_attend(s):
    """Every segment over all its tokens, one by one."""
    c = s.case
    P, G, D, H = c["page"], c["group"], c["dim"], c["heads"]
    ptr, last, q = s.indptr.tolist(), s.last.tolist(), s.q.double().view(-1, G, D)

    def segment(i):
        rows = s.indices[ptr[i]:ptr[i + 1]].long()
        n = (rows.numel() - 1) * P + last[i]
        first = max(0, n - c["window"]) if c["window"] else 0
        k, v = (_values(_bytes(p)[rows].view(p.dtype), s.scales[rows], j).view(-1, D)[first:n]
                for j, p in enumerate((s.k_cache, s.v_cache)))
        x = (k @ q[i].t().contiguous()).t() * D ** -0.5
        if c["cap"]:
            x = torch.tanh(x / c["cap"]) * c["cap"]
        if s.slopes is not None:
            h = i % H
            x = x + s.slopes[h * G:(h + 1) * G, None].double() * torch.arange(first - n + 1, 1, device="cuda")
        return torch.softmax(x, dim=-1) @ v

    return torch.stack([segment(i) for i in range(len(last))]).view(s.q.shape)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "pages": _exact_pages,
            "attend": _exact_attend}[case["kind"]](s)
