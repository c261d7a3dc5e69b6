"""The 8-bit paged cache: append, read-back, page reductions, and decode attention
over it, against the formulas in 64 bits; their refusals; a decode step of all.

Tolerance of the attention, from the arithmetic, for stored values (which are
exact): a score's products are exact in fp32 and their sum off by D 2^-23 sum |q k|,
what follows it by 2^-22 of it, a cap by 2^-20 cap; a weight is off by that as its
logarithm, by 2^-22 (the exponential) and 2^-16 (its two bf16 parts), and an output
by twice the largest such error times sum p |v| / sum p, by T 2^-24 of that (the
accumulation), and by its own rounding, half a step.  With queries of zero and
int8 codes under one exponent every weight is one and every sum exact: those
cases see a single wrong token."""
import ctypes
import math
import random

import pytest
import torch

from vortex_torch import _hip
from vortex_torch.abs import FORMAT, as_vtensor
from vortex_torch.cache import (Context, L2Norm, Max, Mean, Min, MultiReduce, quantized_pool, read_kv_buffer_quant,
                                set_kv_buffer_launcher, set_kv_buffer_quant)
from vortex_torch.decode_attention import (dense_quant_decode_attention, quant_paged_decode_attention,
                                           sparse_quant_decode_attention)
from vortex_torch.utils import ReduceType

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
CODES = [E4M3, INT8]
MOST = {E4M3: 448.0, INT8: 127.0}


# ---------------------------------------------------------------- the format
def _stored(x, codes):
    """(values of the codes, exponent bytes) of rows x, by the definition, in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 128):  # the least e >= -126 with top <= most 2^e
        e = torch.where(top > MOST[codes] * 2.0 ** k, k + 1.0, e)
    y = x * torch.exp2(-e)[..., None]
    if codes == INT8:
        c = torch.round(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        c = torch.round(y / step) * step
    bad = ~torch.isfinite(top)
    return torch.where(bad[..., None], 0.0, c), torch.where(bad, 255, e + 127).to(torch.int64)


def _values(codes, b):
    """Rows of codes with exponent bytes b [...], in 64 bits."""
    f = torch.exp2(b.double() - 127)
    f = torch.where(b == 255, math.nan, torch.where(b == 0, 0.0, f))
    return codes.double() * f[..., None]


def _random_pool(rows, P, D, codes, gen, device, spread=3):
    """Pools of random codes (no NaN) and exponents."""
    if codes == INT8:
        k, v = (torch.randint(-127, 128, (rows, P, D), generator=gen, dtype=torch.int8) for _ in range(2))
    else:
        k, v = (torch.randn((rows, P, D), generator=gen).mul(100).clamp(-448, 448).to(E4M3) for _ in range(2))
    low = 119 if codes == INT8 else 118
    scales = torch.randint(low - spread, low + spread + 1, (rows, P, 2), generator=gen, dtype=torch.uint8)
    return k.to(device), v.to(device), scales.to(device)


def _rows_in(n, H, D, dtype, layout, gen, device):
    randn = lambda *s: torch.randn(s, generator=gen).to(dtype).to(device)  # noqa: E731
    if layout == "fused":
        return [t.unflatten(1, (-1, D)) for t in randn(n, 4 * H * D).split([2 * H * D, H * D, H * D], dim=1)][1:]
    if layout == "heads_first":
        return [randn(H, n, D).transpose(0, 1) for _ in range(2)]
    if layout == "odd":
        return [randn(n, H, D + 1)[..., 1:] for _ in range(2)]
    return [randn(n, H, D) for _ in range(2)]


def _check_append(n, H, D, P, dtype, codes, layout, device, k=None, v=None):
    gen = torch.Generator().manual_seed(n * 31 + D)
    if k is None:
        k, v = _rows_in(n, H, D, dtype, layout, gen, device)
    pages = -(-n // P) + 3
    loc = torch.randperm(pages * P, generator=gen)[:n].to(device)
    if n > 3:
        loc[n - 1], loc[1] = -1, pages * P + 3
    kc, vc, sc = _random_pool(pages * H, P, D, codes, gen, device)
    want = [t.view(torch.uint8).clone() for t in (kc, vc, sc)]
    set_kv_buffer_quant(kc, vc, sc, k, v, loc, P)
    ok = (loc >= 0) & (loc < pages * P)
    at = loc[ok]
    for i, (pool, x) in enumerate(((kc, k), (vc, v))):
        c, b = _stored(x[ok], codes)
        got = pool.view(torch.uint8).view(pages, H, P, D)[at // P, :, at % P].view(codes)
        assert torch.equal(got.double(), c)
        assert torch.equal(sc.view(pages, H, P, 2)[at // P, :, at % P, i].long(), b)
        want[i].view(pages, H, P, D)[at // P, :, at % P] = got.view(torch.uint8)
        want[2].view(pages, H, P, 2)[at // P, :, at % P, i] = b.to(torch.uint8)
    for t, w in zip((kc, vc, sc), want):  # every other row as it was
        assert torch.equal(t.view(torch.uint8), w)
    out = read_kv_buffer_quant(kc, vc, sc, loc, P, H, dtype=dtype)
    for i, (pool, got) in enumerate(zip((kc, vc), out)):
        stored = pool.view(torch.uint8).view(pages, H, P, D)[at // P, :, at % P].view(codes)
        full = _values(stored, sc.view(pages, H, P, 2)[at // P, :, at % P, i].long()).to(dtype)
        assert torch.equal(got[ok].isnan(), full.isnan())
        assert torch.equal(got[ok].nan_to_num(7.0), full.nan_to_num(7.0))
        assert int(got[~ok].count_nonzero()) == 0


SHAPES = [  # tokens, heads, head_dim, page
    (1, 1, 1, 1), (1, 8, 128, 16), (5, 2, 7, 16), (6, 2, 64, 16), (9, 3, 80, 8), (33, 1, 8, 64), (70, 2, 128, 32),
    (7, 3, 256, 5), (257, 1, 96, 64), (4, 2, 512, 16), (3, 2, 576, 16), (40, 5, 100, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_append_and_read(gpu, shape, dtype, codes):
    for layout in ("fused", "apart", "heads_first", "odd"):
        _check_append(*shape, dtype, codes, layout, gpu)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 100])
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_append_of_rows_at_the_borders(gpu, dtype, codes, D):
    """Rows of zeros, of one value, of the smallest and largest ones, at the codes'
    largest and a step past it, on ties, with infinities and NaN."""
    fin = torch.finfo(dtype)
    rows = [torch.zeros(D), torch.full((D,), -0.0)]
    for top in (MOST[codes], MOST[codes] / 2, MOST[codes] * 4, 1.0, 255.0, 1.984375, 1.75):
        for step in (1 - fin.eps, 1.0, 1 + fin.eps):
            rows.append(torch.linspace(-1, 1, D) * top * step)
            rows[-1][D // 2] = top * step
    ties = torch.arange(D) % 64 + 0.5  # halves between whole codes, and between e4m3 steps of 16 to 32
    ties[0] = MOST[codes]
    rows += [ties, -ties, ties / 4]
    for tiny in (fin.tiny, fin.smallest_normal * 2 ** -5, fin.tiny * 3, 2.0 ** -126):
        rows.append(torch.arange(D) % 3 * tiny)
    rows.append(torch.linspace(-1, 1, D) * min(fin.max, 2.0 ** 126))
    for i, odd in enumerate((math.inf, -math.inf, math.nan, -math.nan)):
        r = torch.randn(D, generator=torch.Generator().manual_seed(i))
        r[(i * 37) % D] = odd
        rows.append(r)
    x = torch.stack(rows).to(dtype).to(gpu)[:, None]
    n = x.shape[0]
    _check_append(n, 1, D, 16, dtype, codes, "", gpu, k=x, v=x.flip(0).contiguous())
    if D == 128:
        wide = torch.zeros((n, 3, D + 1), dtype=dtype, device=gpu)  # the element-wide kernel
        wide[:, :, 1:] = x
        _check_append(n, 3, D, 16, dtype, codes, "", gpu, k=wide[..., 1:], v=wide[..., 1:])


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_read_of_every_code_and_exponent(gpu, codes, dtype):
    """256 codes x 256 bytes; NaN codes of e4m3 read as NaN."""
    rows = torch.arange(256, device=gpu, dtype=torch.uint8).expand(256, 1, 256).contiguous()
    b = torch.arange(256, device=gpu, dtype=torch.uint8)
    sc = torch.stack([b, b.flip(0)], -1).view(256, 1, 2)
    zero = (sc == 255) | (sc == 0)
    keep = ~zero.any(-1).view(-1)
    loc = torch.arange(256, device=gpu)
    pool = rows.view(codes)
    k, v = read_kv_buffer_quant(pool, pool.clone(), sc.view(torch.float8_e8m0fnu), loc, 1, 1, dtype=dtype)
    for got, bytes_ in ((k, sc[..., 0]), (v, sc[..., 1])):
        c = pool.view(256, 256).double()
        # in fp32 first, as the kernel's product (past its range an infinity, among its smallest values rounded)
        want = (c * torch.exp2(bytes_.double() - 127)).float().to(dtype)
        assert torch.equal(got[:, 0][keep].isnan(), want[keep].isnan())
        assert torch.equal(got[:, 0][keep].nan_to_num(3.0), want[keep].nan_to_num(3.0))
    finite = pool.view(256, 256)[0].double().isfinite()
    assert int(k[0, 0][finite].count_nonzero()) == 0  # byte 0


@pytest.mark.gpu
def test_read_into_strided_tensors_and_past_the_pool(gpu):
    gen = torch.Generator().manual_seed(5)
    kc, vc, sc = _random_pool(6 * 2, 16, 128, INT8, gen, gpu)
    loc = torch.tensor([3, -1, 95, 96, (1 << 63) - 1, -(1 << 63), 0, 3], device=gpu)
    want = read_kv_buffer_quant(kc, vc, sc, loc, 16, 2)
    both = torch.full((8, 5, 128), 9.0, dtype=torch.bfloat16, device=gpu)
    k, v = read_kv_buffer_quant(kc, vc, sc, loc, 16, 2, k_out=both[:, :2], v_out=both[:, 2:4])
    assert torch.equal(both[:, :2], want[0]) and torch.equal(both[:, 2:4], want[1]) and bool((both[:, 4] == 9).all())
    assert int(want[0][[1, 3, 4, 5]].count_nonzero()) == 0 and torch.equal(want[0][0], want[0][7])
    empty = read_kv_buffer_quant(kc, vc, sc, loc[:0], 16, 2, dtype=torch.float32)
    assert empty[0].shape == empty[1].shape == (0, 2, 128)
    set_kv_buffer_quant(kc, vc, sc, empty[0], empty[1], loc[:0], 16)


@pytest.mark.gpu
@pytest.mark.parametrize("H,P,D", [(1, 16, 128), (3, 5, 7), (8, 16, 64)])
def test_append_slots_far_past_the_pool(gpu, H, P, D):
    pages, guard = 7, 130 * H * P
    far = [pages * P, (1 << 31) - 1, 1 << 32, (1 << 63) // H - 1, (1 << 63) - 1, *(1 << b for b in range(57, 63)),
           *((1 << b) + 3 * P + 2 for b in range(57, 63)), -1, -(1 << 63)]
    loc = torch.tensor([pages * P - 1, *(min(x, (1 << 63) - 1) for x in far)], device=gpu)
    buffers = torch.full((2, guard + pages * H * P + guard, D), 7, dtype=torch.int8, device=gpu)
    scales = torch.full((guard + pages * H * P + guard, 2), 7, dtype=torch.uint8, device=gpu)
    kc, vc = (b[guard:-guard].view(pages * H, P, D) for b in buffers)
    sc = scales[guard:-guard].view(pages * H, P, 2)
    k = torch.randn((loc.numel(), H, D), device=gpu)
    set_kv_buffer_quant(kc, vc, sc, k, k, loc, P)
    c, b = _stored(k[0], INT8)
    assert torch.equal(kc.view(pages, H, P, D)[-1, :, -1].double(), c)
    assert torch.equal(sc.view(pages, H, P, 2)[-1, :, -1, 1].long(), b)
    for t in (kc, vc, sc):
        t.view(pages, H, P, -1)[-1, :, -1] = 7
    assert bool((buffers == 7).all()) and bool((scales == 7).all())
    out = torch.zeros((pages * H, 1, D), dtype=torch.bfloat16, device=gpu)
    _hip.page_reduce_quant(kc, sc, False, [out], [_hip.REDUCE_MAX], loc, H, P, 1)  # closes the pool's last page only
    assert int(out[:-H].count_nonzero()) == 0 and int(out[-H:].count_nonzero()) == H * D


# ---------------------------------------------------------- page reductions
def _context(pages, H, P, D, n):
    ctx = Context()
    ctx.page_size, ctx.head_num, ctx.head_dim, ctx.total_num_pages, ctx.max_new_tokens_per_batch = P, H, D, pages, n
    ctx.profile()
    return ctx


def _paged(t):
    return as_vtensor(t, FORMAT.PAGED)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("H,P,D", [(8, 16, 128), (2, 16, 64), (1, 64, 256), (3, 5, 128), (2, 1, 64), (1, 33, 512),
                                   (2, 16, 80), (1, 7, 3), (2, 16, 576)])
def test_page_reductions_are_those_of_a_bf16_pool(gpu, H, P, D, codes):
    gen = torch.Generator().manual_seed(P + D)
    pages = 23
    kc, vc, sc = _random_pool(pages * H, P, D, codes, gen, gpu)
    loc = torch.cat([torch.arange(4 * P, 9 * P), torch.tensor([3 * P - 1, 11 * P + P // 2, -1, pages * P + P - 1]),
                     torch.tensor([(pages - 1) * P + P - 1])])[torch.randperm(5 * P + 5, generator=gen)].to(gpu)
    types = [ReduceType.Mean, ReduceType.Max, ReduceType.Min, ReduceType.L2Norm]
    same = D in (64, 128, 256, 512)
    for values, pool in ((False, kc), (True, vc)):
        x = quantized_pool(pool, sc, values=values)
        plain = _values(pool, sc[..., int(values)].long()).bfloat16()
        old = torch.randn((pages * H, 1, D), generator=gen).bfloat16().to(gpu)
        for op, rt in ((Mean, 0), (Max, 1), (Min, 2), (L2Norm, 3)):
            for out_type in (torch.bfloat16, torch.float32):
                got, want = old.to(out_type), old.to(out_type)
                ctx = _context(pages, H, P, D, loc.numel())
                a, b = op(dim=1), op(dim=1)
                for o, src, dst in ((a, x, got), (b, _paged(plain), want)):
                    o(src, _paged(dst), loc=loc, ctx=ctx)
                ctx.execute()
                a(x, _paged(got), loc=loc, ctx=ctx)
                b(_paged(plain), _paged(want), loc=loc[(loc >= 0) & (loc < pages * P)].contiguous(), ctx=ctx)
                if same or rt in (1, 2):
                    assert torch.equal(got, want)
                else:  # sums of P terms in another order: P 2^-24 of their sizes, and a rounding each
                    size = plain.double().abs().mean(1, keepdim=True) if rt == 0 else want.double().abs()
                    off = 2 * (P * 2.0 ** -23 * size + 2.0 ** -8 * want.double().abs())
                    assert bool(((got.double() - want.double()).abs() <= off).all())
        outs = [old.clone() for _ in types]
        multi, ctx = MultiReduce(types), _context(pages, H, P, D, loc.numel())
        multi(x, [_paged(o) for o in outs], loc=loc, ctx=ctx)
        ctx.execute()
        multi(x, [_paged(o) for o in outs], loc=loc, ctx=ctx)
        for o, rt in zip(outs, types):
            alone = old.clone()
            _hip.page_reduce_quant(pool, sc, values, [alone], [int(rt.value)], loc, H, P, 1)
            assert torch.equal(o, alone)


@pytest.mark.gpu
def test_page_reductions_of_many_pages_and_of_rows_that_are_no_numbers(gpu):
    gen = torch.Generator().manual_seed(8)
    H, P, D, pages = 8, 16, 128, 2100
    kc, vc, sc = _random_pool(pages * H, P, D, E4M3, gen, gpu)
    loc = torch.arange(pages * P, device=gpu)
    out = torch.zeros((2, pages * H, 1, D), dtype=torch.bfloat16, device=gpu)
    want = torch.zeros_like(out)
    _hip.page_reduce_quant(kc, sc, False, list(out), [_hip.REDUCE_MAX, _hip.REDUCE_MIN], loc, H, P, 1)
    plain = _values(kc, sc[..., 0].long()).bfloat16()
    _hip.page_reduce_multi(plain, list(want), [_hip.REDUCE_MAX, _hip.REDUCE_MIN], loc, H, P, 1)
    assert torch.equal(out, want)
    for t in (_hip.REDUCE_MEAN, _hip.REDUCE_L2NORM):
        _hip.page_reduce_quant(kc, sc, False, [out[0]], [t], loc, H, P, 1)
        _hip.page_reduce(plain, want[0], loc, H, P, 1, t)
        assert torch.equal(out[0], want[0])
    x = torch.randn((1, H, D), device=gpu)
    x[0, 3, 5] = math.inf
    set_kv_buffer_quant(kc, vc, sc, x, x, torch.tensor([40], device=gpu), P)
    mean = torch.zeros((pages * H, 1, D), dtype=torch.bfloat16, device=gpu)
    _hip.page_reduce_quant(kc, sc, False, [mean], [_hip.REDUCE_MEAN], loc, H, P, 1)
    bad = mean.isnan().view(pages, H, D)
    assert bool(bad[2, 3].all()) and int(bad.sum()) == D


# ---------------------------------------------------------------- attention
def _table(tokens, P, H, seed, spare=5, scrambled=False):
    """(indptr, indices, last, pool pages) of requests of so many tokens (0: no pages)."""
    r = random.Random(seed)
    total = sum(-(-t // P) for t in tokens) + spare
    free = list(range(total))
    r.shuffle(free)
    indptr, indices, last = [0], [], []
    for t in tokens:
        mine = [free.pop() for _ in range(-(-t // P))]
        for h in range(H):
            order = sorted(mine, key=lambda p: (p * 7 + h * 13) % 31) if scrambled else mine
            indices += [p * H + h for p in order]
            indptr.append(len(indices))
            last.append((t - 1) % P + 1 if t else 0)
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (indptr, indices, last)) + (total,)


def _plain(q, kc, vc, sc, indptr, indices, last, B, H, scale=None, cap=0.0, window=0, slopes=None):
    """(o, bound) [B * H, G, D] in 64 bits on the CPU, with what the fp32 steps may be off."""
    D, P = kc.shape[2], kc.shape[1]
    rows_of = kc.shape[0]
    q = q.cpu().double().reshape(B * H, -1, D)
    G = q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o, off = torch.zeros((2, B * H, G, D), dtype=torch.float64)
    for s in range(B * H):
        pages = indices[indptr[s]:indptr[s + 1]].long()
        n = (pages.numel() - 1) * P + int(last[s]) if pages.numel() else 0
        seen = torch.arange(max(n, 0))
        seen = seen[(seen >= n - window) | (window <= 0)]
        ok = ((pages >= 0) & (pages < rows_of))[seen // P] if n > 0 else torch.zeros(0, dtype=torch.bool)
        seen = seen[ok]
        if not seen.numel():
            continue
        at = pages[seen // P] * P + seen % P
        there = at.to(kc.device)
        k, v = (_values(t.view(torch.uint8).view(-1, D)[there].view(t.dtype),
                        sc.view(torch.uint8).view(-1, 2)[there, i].long()).cpu() for i, t in enumerate((kc, vc)))
        y = q[s] @ k.t() * scale
        size = q[s].abs() @ k.abs().t() * abs(scale)
        x = cap * torch.tanh(y / cap) if cap else y
        bias = torch.zeros(G, 1)
        if slopes is not None:
            bias = slopes.cpu().double().view(H, G)[s % H][:, None] * (n - 1 - seen)
        x = x - bias
        p = torch.softmax(x, -1)
        e = (D * 2.0 ** -23 * size + 2.0 ** -22 * (y.abs() + bias + 1) + 2.0 ** -20 * cap).amax(-1)
        p_v = p @ v.abs()
        o[s] = p @ v
        off[s] = (2 * e[:, None].expm1() + 2.0 ** -16 + seen.numel() * 2.0 ** -24) * p_v
    return o, off


def _near(got, want, off):
    half = torch.finfo(got.dtype).eps / 2
    got = got.cpu().double().reshape(want.shape)
    bound = off + half * (want.abs() + off) + torch.finfo(torch.float16).smallest_normal * 2.0 ** -11
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


def _case(tokens, H, G, D, P, codes, dtype, device, seed=0, scrambled=False, std=1.0, **kw):
    gen = torch.Generator().manual_seed(seed + D + G)
    indptr, indices, last, pages = _table(tokens, P, H, seed, scrambled=scrambled)
    kc, vc, sc = _random_pool(pages * H, P, D, codes, gen, device)
    B = len(tokens)
    q = (torch.randn((B, H * G, D), generator=gen) * std).to(dtype).to(device)
    tables = [t.to(device) for t in (indptr, indices, last)]
    got = quant_paged_decode_attention(q, kc, vc, sc, *tables, B, H, **kw)
    assert got.shape == q.shape and got.dtype == dtype
    plain = dict(scale=kw.get("sm_scale"), cap=kw.get("logits_soft_cap") or 0.0, window=kw.get("window") or 0,
                 slopes=kw.get("slopes"))
    want, off = _plain(q, kc, vc, sc, indptr, indices, last, B, H, **plain)
    _near(got, want, off)
    return q, kc, vc, sc, indptr, indices, last, got, want, off


RAGGED = [1, 16, 0, 17, 31, 32, 33, 127, 128, 129, 300, 0, 1000]


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 7, 8, 16])
def test_attention_heads_and_types(gpu, G, D, dtype, codes):
    _case(RAGGED, 2, G, D, 16, codes, dtype, gpu, seed=G)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("P", [1, 2, 5, 8, 16, 24, 32, 48, 64, 100, 256])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_pages(gpu, D, P, codes):
    _case([P, 1, 3 * P + 1, 0, 257, 2 * P, 700, P + P // 2 + 1], 3, 4, D, P, codes, torch.bfloat16, gpu, seed=P,
          scrambled=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D,P", [(64, 16), (128, 16), (256, 32), (128, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("kw", [dict(logits_soft_cap=5.0), dict(logits_soft_cap=30.0, sm_scale=1.0),
                                dict(window=1), dict(window=16), dict(window=17), dict(window=100), dict(window=999),
                                dict(window=1 << 30), dict(window=0x7fffffff), dict(slopes=True),
                                dict(slopes=True, window=50, logits_soft_cap=20.0), dict(sm_scale=0.0),
                                dict(sm_scale=-0.3)], ids=str)
def test_attention_caps_windows_and_slopes(gpu, kw, dtype, D, P):
    H, G = 2, 4
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = torch.exp2(-torch.arange(H * G, dtype=torch.float32)).to(gpu)
    _case(RAGGED, H, G, D, P, E4M3 if D == 128 else INT8, dtype, gpu, seed=3, **kw)


def _uniform(tokens, H, G, D, P, device, window=0, codes_seed=1):
    """Queries of zero, one exponent: every output is an exact mean of whole codes."""
    gen = torch.Generator().manual_seed(codes_seed)
    indptr, indices, last, pages = _table(tokens, P, H, codes_seed)
    kc, vc, sc = _random_pool(pages * H, P, D, INT8, gen, device)
    sc.fill_(127)
    B = len(tokens)
    q = torch.zeros((B, H * G, D), dtype=torch.bfloat16, device=device)
    got = quant_paged_decode_attention(q, kc, vc, sc, indptr.to(device), indices.to(device), last.to(device), B, H,
                                       window=window).view(B * H, G, D)
    rows = vc.view(-1, D).cpu().long()
    for s in range(B * H):
        t = tokens[s // H]
        if not t:
            assert int(got[s].count_nonzero()) == 0
            continue
        seen = torch.arange(max(0, t - window) if window else 0, t)
        at = indices[indptr[s]:indptr[s + 1]].long()[seen // P] * P + seen % P
        mean = rows[at].sum(0).double() / seen.numel()
        # the quotient by two fp32 steps, then half a step
        assert bool(((got[s].cpu().double() - mean).abs() <= mean.abs() * (2.0 ** -8 + 2.0 ** -20)).all()), s
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,H,D,P,window", [
    ([20000], 1, 128, 16, 0), ([5000, 3, 0, 40000], 2, 64, 16, 0), ([17, 2000] * 40, 8, 128, 16, 0),
    ([1] * 700, 4, 64, 16, 0), ([5, 0, 64] * 500, 2, 128, 32, 0), ([40000, 9], 1, 256, 64, 0),
    ([9000, 1], 2, 128, 1, 0),
    ([20000, 30, 0, 7000], 2, 128, 16, 1000), ([3000] * 30, 4, 64, 16, 33), ([700, 9000], 1, 256, 5, 4096),
    ([20000, 30, 0, 7000], 2, 128, 16, 3001), ([3000, 1, 0, 1600] * 8, 4, 64, 16, 1500),
    ([0, 9000, 0], 2, 64, 48, 8000),
    ([5000, 0, 9000, 40] * 8, 8, 64, 24, 2500), ([16, 2000] * 150, 1, 128, 16, 2049),
    ([100] * 300 + [30000, 0, 5000], 2, 64, 16, 0), ([100] * 300 + [0, 9000], 2, 128, 5, 0),
    ([3, 40000] + [90] * 500, 1, 256, 16, 0),
    ([0, 0, 0], 2, 64, 16, 0), ([32769], 1, 64, 16, 0)], ids=lambda x: str(x)[:20])
def test_attention_counts_every_token_once(gpu, tokens, H, D, P, window):
    _uniform(tokens, H, 2, D, P, gpu, window=window)


@pytest.mark.gpu
def test_attention_of_many_segments(gpu):
    """More segments than are looked through one by one, some of them empty."""
    r = random.Random(4)
    _uniform([r.choice([0, 1, 15, 16, 40, 200]) for _ in range(1500)], 2, 1, 64, 16, gpu)
    _uniform([r.choice([0, 1, 300, 6000]) for _ in range(1100)], 1, 1, 64, 64, gpu, window=5000)
    _uniform([r.choice([0, 1, 300, 600]) for _ in range(1100)], 1, 1, 64, 5, gpu, window=4500)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(max_tokens=128), dict(max_tokens=1), dict(window=70),
                                dict(max_tokens=100, logits_soft_cap=20.0, slopes=True)], ids=str)
@pytest.mark.parametrize("G,D,P,dtype", [(1, 64, 16, torch.bfloat16), (16, 128, 32, torch.float16),
                                         (5, 256, 16, torch.bfloat16), (3, 256, 64, torch.float16)])
def test_attention_of_many_tiny_segments(gpu, G, D, P, dtype, kw):
    """... a few long ones among them, whatever the caller says of their length."""
    r = random.Random(D + P)
    tokens = [r.choice([0, 1, 7, 16, 17, 32, 33, 64]) for _ in range(530)]
    for i, n in ((0, 129), (1, 513), (200, 2500), (529, 1040)):
        tokens[i] = n
    slopes = torch.rand(2 * G, generator=torch.Generator().manual_seed(G)).to(gpu) if kw.get("slopes") else None
    _case(tokens, 2, G, D, P, E4M3, dtype, gpu, seed=G, **{**kw, "slopes": slopes})


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,H,G,D,P", [
    ([40000], 1, 16, 128, 16), ([40000], 1, 3, 64, 16), ([9000], 1, 1, 64, 8), ([20000], 1, 11, 256, 16),
    ([17000, 30], 2, 5, 128, 32), ([12000, 0, 9000], 1, 9, 256, 64), ([5000] * 6, 2, 16, 64, 16)])
def test_attention_of_few_segments_in_many_parts(gpu, tokens, H, G, D, P):
    """... which several workgroups each join some heads and columns of."""
    _case(tokens, H, G, D, P, E4M3, torch.bfloat16, gpu, seed=len(tokens))


@pytest.mark.gpu
@pytest.mark.parametrize("H,tokens", [(8, [512] * 64), (2, [700] * 3), (3, [5, 900, 0, 33])])
def test_attention_with_a_known_bound(gpu, H, tokens):
    """max_tokens steers how the work is divided, also where it is wrong."""
    for most in (None, 1, max(tokens), 1 << 40):
        _case(tokens, H, 2, 128, 16, E4M3, torch.bfloat16, gpu, max_tokens=most)


@pytest.mark.gpu
@pytest.mark.parametrize("D,P", [(128, 16), (64, 8)])
def test_attention_without_scratch_and_with_it(gpu, D, P):
    """No workspace: a workgroup per segment; the same values."""
    H, G = 2, 4
    q, kc, vc, sc, indptr, indices, last, got, want, off = _case([900, 3, 0, 5000], H, G, D, P, E4M3, torch.bfloat16,
                                                                 gpu)
    B = 4
    lib = _hip.load_library()
    out = torch.full_like(q, 7.0)
    tables = [t.to(gpu) for t in (indptr, indices, last)]
    strides = (ctypes.c_int64 * 3)(H * G * D, G * D, D)

    def call(window, ws, n):
        return lib.vtx_quant_decode_attention(
            q.data_ptr(), strides, out.data_ptr(), kc.data_ptr(), vc.data_ptr(), sc.data_ptr(), kc.shape[0],
            tables[0].data_ptr(), tables[1].data_ptr(), tables[1].numel(), tables[2].data_ptr(), B, H, G, D, P, 0, 0,
            D ** -0.5, 0.0, window, None, 0, ws, n, torch.cuda.current_stream().cuda_stream)

    assert call(0, None, 0) == 0
    _near(out, want, off)
    assert call(40, None, 0) == 0
    _near(out, *_plain(q, kc, vc, sc, indptr, indices, last, B, H, window=40))
    ws = torch.full((4096,), math.nan, device=gpu)
    assert call(0, ws.data_ptr(), ws.numel()) == -1 and b"workspace" in lib.vtx_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 8])
def test_attention_unseen_slots_may_hold_anything(gpu, P):
    """NaN codes, exponents of 255 and 0 behind the last token and in other pages."""
    H, G, D, tokens = 2, 3, 128, [P + 3, 5, 200, 1]
    gen = torch.Generator().manual_seed(2)
    indptr, indices, last, pages = _table(tokens, P, H, 2)
    kc, vc, sc = _random_pool(pages * H, P, D, E4M3, gen, gpu)
    q = torch.randn((4, H * G, D), generator=gen).bfloat16().to(gpu)
    seen = torch.zeros((pages * H, P), dtype=torch.bool)
    for s in range(4 * H):
        rows = indices[indptr[s]:indptr[s + 1]].long()
        seen[rows] = True
        seen[rows[-1], int(last[s]):] = False
    want, off = _plain(q, kc, vc, sc, indptr, indices, last, 4, H)
    for byte in (255, 0, 200):
        for t in (kc, vc):
            t.view(torch.uint8)[~seen.to(gpu)] = 0x7F
        sc[~seen.to(gpu)] = byte
        got = quant_paged_decode_attention(q, kc, vc, sc, indptr.to(gpu), indices.to(gpu), last.to(gpu), 4, H)
        _near(got, want, off)
        windowed = quant_paged_decode_attention(q, kc, vc, sc, indptr.to(gpu), indices.to(gpu), last.to(gpu), 4, H,
                                                window=7)
        _near(windowed, *_plain(q, kc, vc, sc, indptr, indices, last, 4, H, window=7))


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16, 5])
def test_attention_of_rows_that_are_no_numbers(gpu, P):
    """A key or value row with an infinity: NaN for the requests that see it, also
    where it is all they see; the others as ever; outside a window nothing."""
    H, G, D, tokens = 1, 2, 64, [40, 300, 1, 700]
    gen = torch.Generator().manual_seed(3)
    for codes in CODES:
        for what in ("key", "value"):
            indptr, indices, last, pages = _table(tokens, P, H, 3)
            kc, vc, sc = _random_pool(pages, P, D, codes, gen, gpu)
            q = torch.randn((4, G, D), generator=gen).bfloat16().to(gpu)
            slots = [int(indices[indptr[s] + t // P]) * P + t % P for s, t in ((1, 100), (2, 0))]
            x = torch.randn((2, 1, D), generator=gen).to(gpu)
            bad = x.clone()
            bad[:, 0, 7] = math.inf
            set_kv_buffer_quant(kc, vc, sc, bad if what == "key" else x, bad if what == "value" else x,
                                torch.tensor(slots, device=gpu), P)
            tables = [t.to(gpu) for t in (indptr, indices, last)]
            got = quant_paged_decode_attention(q, kc, vc, sc, *tables, 4, 1)
            assert bool(got[1:3].isnan().all())
            want, off = _plain(q, kc, vc, sc, indptr, indices, last, 4, 1)
            _near(got[[0, 3]], want[[0, 3]], off[[0, 3]])
            near = quant_paged_decode_attention(q, kc, vc, sc, *tables, 4, 1, window=150)
            want, off = _plain(q, kc, vc, sc, indptr, indices, last, 4, 1, window=150)
            _near(near[[0, 1, 3]], want[[0, 1, 3]], off[[0, 1, 3]])
            assert bool(near[2].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,P", [(128, 16), (64, 16), (128, 3)])
def test_attention_of_malformed_tables(gpu, D, P):
    """Entries outside the pool count as no tokens, ranges outside the table as no
    pages, last lengths are cut to a page; a table that decreases touches nothing
    outside its buffers."""
    H, G, tokens = 2, 2, [P * 4, 3, 500, 0, 60]
    gen = torch.Generator().manual_seed(9)
    indptr, indices, last, pages = _table(tokens, P, H, 9)
    kc, vc, sc = _random_pool(pages * H, P, D, INT8, gen, gpu)
    q = torch.randn((5, H * G, D), generator=gen).bfloat16().to(gpu)
    run = lambda *t: quant_paged_decode_attention(q, kc, vc, sc, *(x.to(gpu) for x in t), 5, H)  # noqa: E731
    bad = indices.clone()
    bad[[0, 5, int(indptr[4]) + 7]] = torch.tensor([-1, pages * H, 1 << 30], dtype=torch.int32)
    _near(run(indptr, bad, last), *_plain(q, kc, vc, sc, indptr, bad, last, 5, H))
    cut = last.clone()
    cut[0], cut[1], cut[4] = -7, 0, 10 * P
    clear = cut.clamp(0, P)
    _near(run(indptr, indices, cut), *_plain(q, kc, vc, sc, indptr, indices, clear, 5, H))
    long = indptr.clone()
    long[-1] += 1000  # the last segment reaches past the table
    want, off = _plain(q, kc, vc, sc, indptr, indices, last, 5, H)
    want[-1], off[-1] = 0, 0
    _near(run(long, indices, last), want, off)
    r = torch.Generator().manual_seed(1)
    for low, high in ((0, indices.numel()), (-(1 << 31), (1 << 31) - 1), (-5, indices.numel() + 5)):
        p = torch.randint(low, high, indptr.shape, generator=r).to(torch.int32)
        assert run(p, indices, last).shape == q.shape
    assert int(run(indptr, indices[:0], last).count_nonzero()) == 0


@pytest.mark.gpu
def test_attention_layouts_of_queries_and_outputs(gpu):
    """[B * H, G, D], slices of a projection, heads first, an output of the caller's, in place."""
    H, G, D, P = 2, 4, 128, 16
    q, kc, vc, sc, indptr, indices, last, got, want, off = _case([100, 1, 900], H, G, D, P, E4M3, torch.float16, gpu)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    run = lambda q, **kw: quant_paged_decode_attention(q, kc, vc, sc, *t, 3, H, **kw)  # noqa: E731
    assert torch.equal(run(q.view(3 * H, G, D)).view(q.shape), got)
    wide = torch.randn((3, H * G * D + 1024), device=gpu).half()
    wide[:, :H * G * D] = q.view(3, -1)
    assert torch.equal(run(wide[:, :H * G * D].unflatten(1, (-1, D))), got)
    assert torch.equal(run(q.transpose(0, 1).contiguous().transpose(0, 1)), got)
    out = torch.empty_like(q)
    assert run(q, out=out) is out and torch.equal(out, got)
    same = q.clone()
    assert torch.equal(run(same, out=same), got)
    one = quant_paged_decode_attention(wide[:1, :H * G * D].unflatten(1, (-1, D)), kc, vc, sc, t[0], t[1], t[2], 1, H)
    _near(one, want[:H], off[:H])
    empty = quant_paged_decode_attention(q[:0], kc, vc, sc, t[0][:1], t[1], t[2][:0], 0, H)
    assert empty.shape == (0, H * G, D)
    e8 = quant_paged_decode_attention(q, kc, vc, sc.view(torch.float8_e8m0fnu), *t, 3, H)
    assert torch.equal(e8, got)


@pytest.mark.gpu
def test_attention_of_a_pool_past_four_gib(gpu):
    H, G, D, P = 1, 2, 128, 16
    pages = (1 << 32) // (P * D) + 40
    kc, vc = (torch.zeros((pages, P, D), dtype=torch.int8, device=gpu) for _ in range(2))
    sc = torch.full((pages, P, 2), 120, dtype=torch.uint8, device=gpu)
    gen = torch.Generator().manual_seed(1)
    loc = torch.cat([torch.arange((pages - 12) * P, pages * P), torch.arange(0, 5 * P)]).to(gpu)
    k, v = (torch.randn((loc.numel(), 1, D), generator=gen).bfloat16().to(gpu) for _ in range(2))
    set_kv_buffer_quant(kc, vc, sc, k, v, loc, P)
    back = read_kv_buffer_quant(kc, vc, sc, loc, P, H)
    assert float((back[0].double() - k.double()).abs().max()) < 0.05
    mean = torch.zeros((pages, 1, D), dtype=torch.bfloat16, device=gpu)
    _hip.page_reduce_quant(kc, sc, False, [mean], [_hip.REDUCE_MEAN], loc[:12 * P].contiguous(), H, P, 1)
    want = back[0][:12 * P].view(12, P, D).double().mean(1)
    assert bool(((mean[-12:, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all())
    indices = torch.cat([torch.arange(pages - 12, pages), torch.arange(5)]).to(torch.int32)
    indptr, last = torch.tensor([0, 17], dtype=torch.int32), torch.tensor([9], dtype=torch.int32)
    q = torch.randn((1, G, D), generator=gen).bfloat16().to(gpu)
    got = quant_paged_decode_attention(q, kc, vc, sc, indptr.to(gpu), indices.to(gpu), last.to(gpu), 1, H)
    _near(got, *_plain(q, kc, vc, sc, indptr, indices, last, 1, H))


@pytest.mark.gpu
def test_streams_graphs_and_repeats(gpu):
    """Captured steps (append, page means, attention) in two graphs replayed in turn
    and beside eager calls, on two streams; a call's bits repeat."""
    H, G, D, P, B = 2, 4, 128, 16, 6
    gen = torch.Generator().manual_seed(6)
    indptr, indices, last, pages = _table([500, 33, 2000, 16, 0, 70], P, H, 6)
    t = [x.to(gpu) for x in (indptr, indices, last)]
    kc, vc, sc = _random_pool(pages * H, P, D, INT8, gen, gpu)
    mean = torch.zeros((pages * H, 1, D), dtype=torch.bfloat16, device=gpu)
    ends = [(int(indptr[b * H]), int(indptr[b * H + H])) for b in range(B)]
    loc = torch.tensor([int(indices[e - 1]) // H * P + P - 1 if e > a else -1 for a, e in ends], device=gpu)
    qs = [torch.randn((B, H * G, D), generator=gen).bfloat16().to(gpu) for _ in range(2)]
    k, v = (torch.randn((B, H, D), generator=gen).bfloat16().to(gpu) for _ in range(2))

    def step(q, out=None):
        set_kv_buffer_quant(kc, vc, sc, k, v, loc, P)
        _hip.page_reduce_quant(kc, sc, False, [mean], [_hip.REDUCE_MEAN], loc, H, P, 1)
        return quant_paged_decode_attention(q, kc, vc, sc, *t, B, H, out=out)

    first = step(qs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [step(qs[0]) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, first) for x in again)
    graphs, outs = [], [torch.empty_like(q) for q in qs]
    for q, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(q, o)
        graphs.append(g)
    for turn in range(3):
        k.copy_(torch.randn((B, H, D), generator=gen).bfloat16())
        t[2][0] = turn + 3
        for q, g, o in zip(qs, graphs, outs):
            mean.zero_()
            g.replay()
            seen = mean.clone()
            eager = step(q)
            torch.cuda.synchronize()
            assert torch.equal(o, eager) and torch.equal(seen, mean)
        with torch.cuda.stream(side):
            graphs[0].replay()
        other = step(qs[1])
        torch.cuda.synchronize()
        assert torch.equal(other, outs[1])


# ------------------------------------------------------------ all together
@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("name", ["block_sparse_attention", "gqa_block_sparse_attention", "gqa_quest_sparse_attention"])
def test_decode_step_of_a_flow_on_an_8_bit_cache(gpu, name, codes):
    """A registered flow, unchanged, on a quantised cache: append, page finish,
    indexer and attention; centroids and selection are bit for bit those of a
    bf16 cache that holds the same values, and the attention that of the pages
    selected."""
    import workloads as W
    from vortex_torch import flow as vflow
    from vortex_torch.indexer.utils_sglang import plan_decode

    batch = W.c1()
    H, G, D, P, B = batch.num_kv_heads, batch.group_size, batch.head_dim, batch.page_size, batch.batch
    rows = batch.pool_pages * H
    raw = W.k_pool(batch, 10, gpu)
    gen = torch.Generator().manual_seed(1)
    L = int(batch.seq_lens[0])
    loc = torch.tensor([int(batch.pages[0][j // P]) * P + j % P for j in range(L)], device=gpu)
    kc, vc = (torch.zeros((rows, P, D), dtype=torch.uint8, device=gpu).view(codes) for _ in range(2))
    sc = torch.full((rows, P, 2), 1, dtype=torch.uint8, device=gpu)
    new_k = raw.view(-1, H, P, D)[loc // P, :, loc % P]
    new_v = torch.randn(new_k.shape, generator=gen).bfloat16().to(gpu)
    set_kv_buffer_quant(kc, vc, sc, new_k, new_v, loc, P)
    k16, v16 = (torch.zeros((rows, P, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    set_kv_buffer_launcher(k16, v16, *(t.contiguous() for t in read_kv_buffer_quant(kc, vc, sc, loc, P, H)), loc, P)
    q = W.randn_bf16((B * H, G, D), 11, gpu)
    found = []
    for keys in (quantized_pool(kc, sc), as_vtensor(k16, FORMAT.PAGED)):
        ictx, cctx = W.make_contexts(batch, gpu)
        flow = vflow.build_vflow(name)
        cache = {"k": keys}
        for n, (d0, d1) in flow.create_cache(P, D).items():
            cache[n] = as_vtensor(torch.zeros((rows, d0, d1), device=gpu, dtype=torch.bfloat16), FORMAT.PAGED)
        tq = as_vtensor(q.clone(), FORMAT.BATCHED)
        o = as_vtensor(ictx.sparse_kv_indices.view(-1, 1, 1), FORMAT.RAGGED)
        for c in (ictx, cctx):
            c.profile()
        flow.forward_cache(cache, loc, cctx)
        flow.forward_indexer(tq, o, cache, ictx)
        for c in (ictx, cctx):
            c.execute()
        b = batch.to(gpu)
        plan_decode(b.seq_lens, b.req_to_token, b.req_indices, ictx)
        for part in (loc, loc[-1:]):  # the prompt, then a decode step whose page closes
            flow.forward_cache(cache, part, cctx)
        flow.forward_indexer(tq, o, cache, ictx)
        torch.cuda.synchronize()
        found.append((ictx, [cache[n].as_subclass(torch.Tensor).clone() for n in flow.create_cache(P, D)]))
    (ictx, stats), (other, plain_stats) = found
    assert all(torch.equal(a, b) for a, b in zip(stats, plain_stats))
    assert torch.equal(ictx.sparse_kv_indices, other.sparse_kv_indices)
    got = sparse_quant_decode_attention(q, kc, vc, sc, ictx)
    tables = [t.cpu() for t in (ictx.sparse_kv_indptr, ictx.sparse_kv_indices, ictx.kv_last_page_len)]
    _near(got, *_plain(q, kc, vc, sc, *tables, B, H))
    full = dense_quant_decode_attention(q, kc, vc, sc, ictx, logits_soft_cap=30.0, window=1000)
    tables = [t.cpu() for t in (ictx.dense_kv_indptr, ictx.dense_kv_indices, ictx.kv_last_page_len)]
    _near(full, *_plain(q, kc, vc, sc, *tables, B, H, cap=30.0, window=1000))


# ------------------------------------------------------------- refusals (CPU)
def _pool_args(**changes):
    n, H, D, P = 3, 2, 16, 8
    a = dict(k_cache=torch.zeros((2 * H, P, D), dtype=INT8), v_cache=torch.zeros((2 * H, P, D), dtype=INT8),
             kv_scales=torch.zeros((2 * H, P, 2), dtype=torch.uint8), new_k=torch.zeros((n, H, D)),
             new_v=torch.zeros((n, H, D)), loc=torch.arange(n), page_size=P)
    a.update(changes)
    return a


_BYTES = torch.zeros(4096, dtype=torch.int8)
_POOL = _BYTES[:512].view(4, 8, 16)


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_hip, "_current_device", lambda: 0)
    monkeypatch.setattr(_hip, "_stream_of", lambda index: 0)


APPEND_REFUSALS = [
    (dict(k_cache=torch.zeros((4, 8, 16), dtype=torch.bfloat16)), "must hold float8_e4m3fn or int8"),
    (dict(k_cache=torch.zeros((4, 8, 16), dtype=torch.uint8)), "must hold float8_e4m3fn or int8"),
    (dict(v_cache=torch.zeros((4, 8, 16), dtype=E4M3)), "of the same codes"),
    (dict(v_cache=torch.zeros((6, 8, 16), dtype=INT8)), "must both be"),
    (dict(kv_scales=torch.zeros((4, 8, 2), dtype=torch.int8)), "kv_scales must be uint8"),
    (dict(kv_scales=torch.zeros((4, 8, 2))), "kv_scales must be uint8"),
    (dict(kv_scales=torch.zeros((4, 8), dtype=torch.uint8)), "kv_scales must be \\(4, 8, 2\\)"),
    (dict(kv_scales=torch.zeros((4, 8, 4), dtype=torch.uint8)[..., ::2]), "must be contiguous"),
    (dict(k_cache=torch.zeros((4, 8, 32), dtype=INT8)[..., :16]), "must be contiguous"),
    (dict(k_cache=_POOL, v_cache=_POOL), "share memory"),
    (dict(k_cache=_POOL, v_cache=_BYTES[511:1023].view(4, 8, 16)), "share memory"),
    (dict(k_cache=_POOL, kv_scales=_BYTES[500:564].view(torch.uint8).view(4, 8, 2)), "share memory"),
    (dict(new_v=torch.zeros((3, 1, 16))), "must both be"),
    (dict(new_v=torch.zeros((3, 2, 16), dtype=torch.bfloat16)), "bfloat16, float16 or float32"),
    (dict(new_k=torch.zeros((3, 2, 16)).double(), new_v=torch.zeros((3, 2, 16)).double()), "bfloat16, float16 or"),
    (dict(new_k=torch.zeros((3, 2, 32))[..., ::2]), "dense rows"),
    (dict(new_k=torch.zeros((3, 2, 8)), new_v=torch.zeros((3, 2, 8))), "must be \\[pages"),
    (dict(new_k=torch.zeros((3, 0, 16)), new_v=torch.zeros((3, 0, 16))), "must have heads"),
    (dict(new_k=torch.zeros((3, 3, 16)), new_v=torch.zeros((3, 3, 16))), "not pages of 3"),
    (dict(page_size=16), "must be \\[pages"),
    (dict(loc=torch.arange(3, dtype=torch.int32)), "loc must be torch.int64"),
    (dict(loc=torch.arange(6)[::2]), "loc must be contiguous"),
    (dict(loc=torch.arange(2)), "shorter"),
    (dict(k_cache=_POOL, new_k=_BYTES[448:832].view(torch.float32).view(3, 2, 16)), "new_k lies in the pools"),
    (dict(v_cache=_BYTES[512:1024].view(4, 8, 16), new_v=_BYTES[192:576].view(torch.float32).view(3, 2, 16)),
     "new_v lies in the pools")]


@pytest.mark.parametrize("changes, says", APPEND_REFUSALS)
def test_append_refusals(no_gpu, changes, says):
    with pytest.raises(RuntimeError, match=says):
        set_kv_buffer_quant(**_pool_args(**changes))


@pytest.mark.parametrize("changes, says", [
    (dict(dtype=torch.float64), "dtype must be"), (dict(num_kv_heads=0), "num_kv_heads must be positive"),
    (dict(num_kv_heads=3), "not pages of 3"), (dict(page_size=4), "must be \\[pages"),
    (dict(k_out=torch.zeros((3, 2, 16))), "go together"),
    (dict(k_out=torch.zeros((2, 2, 16)), v_out=torch.zeros((2, 2, 16))), "k_out must be \\[3, 2"),
    (dict(k_out=torch.zeros((3, 2, 16)), v_out=torch.zeros((3, 2, 16)).half()), "must both be bfloat16"),
    (dict(k_out=torch.zeros((1, 2, 16)).expand(3, 2, 16), v_out=torch.zeros((3, 2, 16))), "rows that share memory"),
    (dict(k_out=_BYTES[1024:1408].view(torch.float32).view(3, 2, 16),
          v_out=_BYTES[1088:1472].view(torch.float32).view(3, 2, 16)), "shares memory"),
    (dict(k_cache=_POOL, k_out=_BYTES[:384].view(torch.float32).view(3, 2, 16), v_out=torch.zeros((3, 2, 16))),
     "k_out lies in the pools"),
    (dict(kv_scales=torch.zeros((4, 8, 3), dtype=torch.uint8)), "kv_scales must be"),
    (dict(loc=torch.zeros(3)), "loc must be torch.int64")])
def test_read_refusals(no_gpu, changes, says):
    a = _pool_args()
    a = dict({n: a[n] for n in ("k_cache", "v_cache", "kv_scales", "loc", "page_size")}, num_kv_heads=2)
    a.update(changes)
    with pytest.raises(RuntimeError, match=says):
        read_kv_buffer_quant(**a)


def test_pool_and_reduction_refusals(no_gpu):
    a = _pool_args()
    with pytest.raises(RuntimeError, match="codes must hold"):
        quantized_pool(a["k_cache"].float(), a["kv_scales"])
    with pytest.raises(RuntimeError, match="kv_scales must be"):
        quantized_pool(a["k_cache"], a["kv_scales"][:2])
    out = torch.zeros((4, 1, 16), dtype=torch.bfloat16)
    call = lambda out=out, types=(0,), loc=a["loc"], P=8, dim=1: _hip.page_reduce_quant(  # noqa: E731
        a["k_cache"], a["kv_scales"], False, [out], types, loc, 2, P, dim)
    for kw, says in ((dict(dim=2), "dim 1"), (dict(P=4), "must be \\[rows, 4"), (dict(out=out.half()), "bf16 or fp32"),
                     (dict(loc=a["loc"].int()), "loc must be"), (dict(types=(0, 1)), "one type each"),
                     (dict(out=out[..., :15].contiguous()), "multiple of its row"),
                     (dict(out=a["k_cache"].view(torch.bfloat16).view(16, 1, 16)), "share memory")):
        with pytest.raises(RuntimeError, match=says):
            call(**kw)
    plain = as_vtensor(a["k_cache"], FORMAT.PAGED)
    assert not hasattr(plain, "_quantized")
    pool = quantized_pool(a["k_cache"], a["kv_scales"], values=True)
    assert pool._format == FORMAT.PAGED and pool.data_ptr() == a["k_cache"].data_ptr()


def _attention_args(**changes):
    B, H, G, D, P = 2, 2, 3, 64, 8
    a = dict(q=torch.zeros((B, H * G, D), dtype=torch.bfloat16), k_cache=torch.zeros((8, P, D), dtype=INT8),
             v_cache=torch.zeros((8, P, D), dtype=INT8), kv_scales=torch.zeros((8, P, 2), dtype=torch.uint8),
             kv_indptr=torch.zeros(B * H + 1, dtype=torch.int32), kv_indices=torch.zeros(8, dtype=torch.int32),
             kv_last_page_len=torch.zeros(B * H, dtype=torch.int32), batch_size=B, num_kv_heads=H)
    a.update(changes)
    return a


@pytest.mark.parametrize("changes, says", [
    (dict(k_cache=torch.zeros((8, 8, 64), dtype=torch.bfloat16)), "must hold"),
    (dict(v_cache=torch.zeros((8, 8, 32), dtype=INT8)), "must both be"),
    (dict(kv_scales=torch.zeros((8, 8, 1), dtype=torch.uint8)), "kv_scales must be"),
    (dict(q=torch.zeros((2, 6, 64))), "bfloat16 or float16"),
    (dict(q=torch.zeros((2, 6, 32), dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros((2, 5, 64), dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros((3, 6, 64), dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros((2, 6, 128), dtype=torch.bfloat16)[..., ::2]), "dense rows"),
    (dict(out=torch.zeros((2, 6, 64), dtype=torch.float16)), "q and out must both"),
    (dict(out=torch.zeros((4, 3, 64), dtype=torch.bfloat16)), "out must be"),
    (dict(out=torch.zeros((2, 6, 128), dtype=torch.bfloat16)[..., :64]), "out must be"),
    (dict(kv_indptr=torch.zeros(4, dtype=torch.int32)), "entries"),
    (dict(kv_last_page_len=torch.zeros(3, dtype=torch.int32)), "entries"),
    (dict(kv_indptr=torch.zeros(5)), "kv_indptr must be"),
    (dict(kv_indices=torch.zeros(16, dtype=torch.int32)[::2]), "kv_indices must be contiguous"),
    (dict(batch_size=-1), "positive"), (dict(num_kv_heads=0), "positive"),
    (dict(logits_soft_cap=-1.0), "logits_soft_cap"), (dict(logits_soft_cap=math.nan), "logits_soft_cap"),
    (dict(logits_soft_cap=math.inf), "logits_soft_cap"),
    (dict(window=-1), "window"), (dict(window=1 << 31), "window"),
    (dict(slopes=torch.zeros(5)), "slopes must be 6"), (dict(slopes=torch.zeros(6).half()), "slopes must be 6"),
    (dict(slopes=torch.zeros(12)[::2]), "slopes must be 6")])
def test_attention_refusals(no_gpu, changes, says):
    with pytest.raises(RuntimeError, match=says):
        quant_paged_decode_attention(**_attention_args(**changes))


def test_calls_need_a_gpu():
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        set_kv_buffer_quant(**_pool_args())
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        quant_paged_decode_attention(**_attention_args())
    a = _pool_args()
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        read_kv_buffer_quant(a["k_cache"], a["v_cache"], a["kv_scales"], a["loc"], 8, 2)


def test_c_refusals():
    lib = _hip.load_library()
    p = [0x10000 * (i + 1) for i in range(12)]
    four, three = (ctypes.c_int64 * 4)(32, 16, 32, 16), (ctypes.c_int64 * 3)(384, 192, 64)

    def rows(f, n=3, H=2, D=16, dtype=0, codes=0, P=8, k=p[0], loc=p[5], sc=p[2]):
        return f(k, p[1], sc, 32, p[3], p[4], four, loc, n, H, D, dtype, codes, P, None)

    for f in (lib.vtx_set_kv_buffer_quant, lib.vtx_read_kv_buffer_quant):
        for kw, says in ((dict(n=-1), b"bad sizes"), (dict(H=0), b"bad sizes"), (dict(D=0), b"bad sizes"),
                         (dict(P=0), b"bad sizes"), (dict(dtype=3), b"element type"), (dict(codes=2), b"codes"),
                         (dict(k=None), b"null"), (dict(loc=None), b"null"), (dict(sc=p[2] + 1), b"2-byte"),
                         (dict(H=1 << 25), b"too many heads")):
            assert rows(f, **kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
        assert rows(f, n=0) == 0

    def reduce(n_out=1, codes=0, P=16, C=64, H=2, nnz=4, x=p[0], out=p[3], dtype=0, rt=0):
        one = (ctypes.c_void_p * 1)(out)
        return lib.vtx_page_reduce_quant(x, p[1], 64, P, C, codes, n_out, one, (ctypes.c_int32 * 1)(dtype),
                                         (ctypes.c_int32 * 1)(rt), 64, p[4], nnz, H, None)

    for kw, says in ((dict(n_out=0), b"1..4"), (dict(n_out=5), b"1..4"), (dict(codes=7), b"codes"),
                     (dict(P=0), b"sizes"), (dict(C=0), b"sizes"), (dict(H=0), b"sizes"), (dict(nnz=-1), b"sizes"),
                     (dict(x=None), b"null"),
                     (dict(out=None), b"null"), (dict(dtype=2), b"dtype"), (dict(rt=4), b"reduce type"),
                     (dict(H=1 << 30), b"too many heads")):
        assert reduce(**kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
    assert reduce(nnz=0) == 0

    def attend(B=2, H=2, G=3, D=64, P=8, dtype=0, codes=0, cap=0.0, window=0, q=p[0], k=p[2], entries=8, st=three,
               longest=0):
        return lib.vtx_quant_decode_attention(q, st, p[1], k, p[3], p[4], 32, p[5], p[6], entries, p[7], B, H, G, D, P,
                                              dtype, codes, 0.1, cap, window, None, longest, None, 0, None)

    for kw, says in ((dict(B=-1), b"sizes"), (dict(H=0), b"sizes"), (dict(P=0), b"sizes"), (dict(window=-1), b"sizes"),
                     (dict(entries=-1), b"sizes"), (dict(longest=-1), b"sizes"), (dict(D=96), b"not supported"),
                     (dict(G=17), b"not supported"),
                     (dict(G=0), b"not supported"), (dict(dtype=1), b"element type"), (dict(codes=2), b"codes"),
                     (dict(cap=-1.0), b"cap"), (dict(cap=math.nan), b"cap"), (dict(cap=math.inf), b"cap"),
                     (dict(q=None), b"null"), (dict(q=p[0] + 8), b"aligned"), (dict(k=p[2] + 4), b"aligned"),
                     (dict(st=(ctypes.c_int64 * 3)(384, 192, 63)), b"aligned"), (dict(entries=1 << 31), b"entries"),
                     (dict(B=1 << 20, H=1 << 12), b"too many"), (dict(B=(1 << 22) + 1), b"too many")):
        assert attend(**kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
    assert attend(B=0) == 0
    need = lib.vtx_quant_decode_attention_workspace_len
    assert need(2, 2, 3, 64, 8, 0, 0, 1 << 20) > 0 and need(0, 2, 3, 64, 8, 0, 0, 1 << 20) == 0
    assert need(2, 2, 17, 64, 8, 0, 0, 1 << 20) == 0
    # where no segment can be long, none is divided
    assert need(2, 2, 3, 64, 8, 0, 0, 8) == 0 and need(2, 2, 3, 64, 8, 0, 300, 1 << 20) == 0
    assert need(2, 2, 3, 64, 8, 300, 0, 1 << 20) == 0 and need(2, 2, 3, 64, 8, 30000, 30000, 1 << 20) > 0
