"""The 8-bit paged cache at the edges of what it accepts, against the formulas and
by the tolerances of test_quant_cache."""
import ctypes
import math
import random

import pytest
import torch

from test_quant_cache import CODES, E4M3, INT8, _case, _near, _plain, _random_pool, _table
from vortex_torch import _hip
from vortex_torch.cache import set_kv_buffer_quant
from vortex_torch.decode_attention import quant_paged_decode_attention


# --------------------------------------------------------------------- caps
@pytest.mark.gpu
@pytest.mark.parametrize("D,P", [(64, 16), (128, 5), (256, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e5, 1e6, 1e9, 1e20, 3e38, 1e39, 1e300])
def test_large_caps(gpu, cap, dtype, D, P):
    """The bound follows the scores, not the cap: that of uncapped ones, whose sum of
    products is allowed D 2^-23 sum |q k|, twice what D fp32 additions are off by.  The
    other half, at least 2^-18 of the score, has room for the cap's steps: 2^-20 of it.
    (Between the two formulas lies y (y / cap)^2 / 3, 2^-19 |y| for |y| <= 2 at 1e3.)"""
    H, G, tokens = 2, 4, [700, 1, 33, 0, 2000]
    gen = torch.Generator().manual_seed(D)
    indptr, indices, last, pages = _table(tokens, P, H, 3)
    kc, vc, sc = _random_pool(pages * H, P, D, E4M3, gen, gpu, spread=1)
    q = (torch.randn((5, H * G, D), generator=gen) * 2.5).to(dtype).to(gpu)
    got = quant_paged_decode_attention(q, kc, vc, sc, *(t.to(gpu) for t in (indptr, indices, last)), 5, H,
                                       logits_soft_cap=cap)
    want, _ = _plain(q, kc, vc, sc, indptr, indices, last, 5, H, cap=cap)
    _, off = _plain(q, kc, vc, sc, indptr, indices, last, 5, H)
    _near(got, want, off)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-3, 1e-20, 1e-37, 1e-40, 1e-46, 1e-300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_small_caps(gpu, dtype, cap):
    """... down to where every score is almost the same, scores of zero among them;
    a cap that fp32 holds as 0 is a cap all the same."""
    H, G, D, P, tokens = 2, 2, 64, 16, [300, 17]
    gen = torch.Generator().manual_seed(1)
    indptr, indices, last, pages = _table(tokens, P, H, 3)
    kc, vc, sc = _random_pool(pages * H, P, D, INT8, gen, gpu)
    q = torch.randn((2, H * G, D), generator=gen).to(dtype).to(gpu)
    q[:, 1] = 0
    got = quant_paged_decode_attention(q, kc, vc, sc, *(t.to(gpu) for t in (indptr, indices, last)), 2, H,
                                       logits_soft_cap=cap)
    # a score is at most the cap, and off by 2^-20 of it
    want, _ = _plain(q, kc, vc, sc, indptr, indices, last, 2, H, cap=cap)
    _, off = _plain(q * 0, kc, vc, sc, indptr, indices, last, 2, H)
    _near(got, want, off + 2.0 ** -19 * cap)


@pytest.mark.gpu
@pytest.mark.parametrize("D,P", [(64, 16), (128, 5), (256, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_an_infinite_query_under_a_cap(gpu, dtype, D, P):
    """Its scores are infinities by the keys' signs, which a cap makes +-cap."""
    H, G, n, cap = 1, 2, 200, 3.0
    gen = torch.Generator().manual_seed(D)
    indptr, indices, last, pages = _table([n], P, H, 3)
    kc, vc, sc = _random_pool(pages * H, P, D, INT8, gen, gpu)
    kc[kc == 0] = 1
    q = torch.randn((1, G, D), generator=gen).to(dtype).to(gpu)
    q[0, :, 7] = torch.tensor([math.inf, -math.inf])
    got = quant_paged_decode_attention(q, kc, vc, sc, *(t.to(gpu) for t in (indptr, indices, last)), 1, H,
                                       logits_soft_cap=cap)
    at = indices.long()[torch.arange(n) // P] * P + torch.arange(n) % P
    sign = kc.view(-1, D).cpu()[at, 7].double().sign()
    v = vc.view(-1, D).cpu()[at].double() * torch.exp2(sc.view(-1, 2).cpu()[at, 1].double() - 127)[:, None]
    p = torch.softmax(torch.stack([sign, -sign]) * cap, -1)
    # +-cap is exact to 2^-20 of it; the weights' and the sums' errors as ever
    off = (2 * math.expm1(2.0 ** -20 * cap + 2.0 ** -22) + 2.0 ** -16 + n * 2.0 ** -24) * (p @ v.abs())
    _near(got, p @ v, off)
    got = quant_paged_decode_attention(q, kc, vc, sc, *(t.to(gpu) for t in (indptr, indices, last)), 1, H)
    assert bool(got.isnan().all())


# ------------------------------------------------------------------ lengths
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_longest_segments_and_longer_ones(gpu, D):
    """Tables of one page over and over: 2^30 - 1024 tokens are attended to (weights of
    one and values of 64, every sum exact), 2^30 give NaN, not the zeros of a segment
    without tokens; those beside them are as ever."""
    P, most = 1024, 1 << 20
    kc, vc, sc = _random_pool(2, P, D, INT8, torch.Generator().manual_seed(1), gpu)
    vc.fill_(64)
    sc.fill_(127)
    q = torch.zeros((3, 2, D), dtype=torch.bfloat16, device=gpu)
    for pages, window, far in ((most, 0, True), (most, 5000, True), (most + 7, 0, True), (most - 1, 0, False)):
        if not far and D != 64:
            continue
        indices = torch.ones(pages + 3, dtype=torch.int32, device=gpu)
        indptr = torch.tensor([0, 2, 2 + pages, 3 + pages], dtype=torch.int32, device=gpu)
        last = torch.tensor([5, P, 9], dtype=torch.int32, device=gpu)
        for known in (None, 100):  # divided over the card, and a workgroup each
            if known and not far:
                continue
            got = quant_paged_decode_attention(q, kc, vc, sc, indptr, indices, last, 3, 1, window=window,
                                               max_tokens=known)
            assert bool((got[[0, 2]] == 64).all())
            assert bool(got[1].isnan().all() if far else (got[1] == 64).all())


# ------------------------------------------------- windows on divided tables
def _windowed(tokens, H, G, D, P, window, codes, dtype, device, **kw):
    need = _hip.load_library().vtx_quant_decode_attention_workspace_len
    entries = H * sum(-(-t // P) for t in tokens)
    assert need(len(tokens), H, G, D, P, window, 0, entries) > 0  # (not a workgroup per segment)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.exp2(-2.0 - torch.arange(H * G, dtype=torch.float32)).to(device)
    _case(tokens, H, G, D, P, codes, dtype, device, seed=window, window=window, **kw)


SCORES = [dict(), dict(slopes=True), dict(logits_soft_cap=2.0), dict(logits_soft_cap=8.0, slopes=True, sm_scale=0.2)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SCORES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("D,P,window", [(64, 16, 1500), (128, 16, 3001), (256, 32, 2050), (128, 5, 1025),
                                        (64, 48, 5000)])
def test_windows_on_a_packed_line(gpu, D, P, window, dtype, kw):
    """Segments cut by ranges and by the window, whose parts have maxima of their own;
    shorter ones and empty ones between them."""
    _windowed([9000, 30, 0, 7001, 1, 2600, window, window + 1, 17], 2, 3, D, P, window, INT8 if D == 64 else E4M3,
              dtype, gpu, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SCORES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("count,D,P,window", [(600, 64, 16, 2500), (300, 256, 16, 1100), (1030, 64, 32, 4200),
                                              (1030, 128, 5, 4500)])
def test_windows_on_tables_of_many_segments(gpu, count, D, P, window, dtype, kw):
    """... packed ones of under 1024 segments, spaced ones of more."""
    r = random.Random(count)
    tokens = [r.choice([0, 1, 16, 33, 200]) for _ in range(count)]
    for i, n in ((0, window + 700), (3, 9000), (count // 2, window), (count - 1, 2 * window + 5)):
        tokens[i] = n
    _windowed(tokens, 1, 2, D, P, window, E4M3, dtype, gpu, **kw)


# ---------------------------------------------------------- malformed tables
@pytest.mark.gpu
def test_overlapping_segments_of_more_parts_than_32_bits_count(gpu):
    """20,000 segments of which every other one is the whole table, 2^25 pages in 2^19
    parts each: nothing is written but the outputs and the workspace."""
    S, D, P, pages = 20000, 64, 16, 1 << 25
    lib = _hip.load_library()
    kc, vc, sc = _random_pool(1, P, D, INT8, torch.Generator().manual_seed(1), gpu)
    indices = torch.zeros(pages, dtype=torch.int32, device=gpu)
    indptr = torch.zeros(S + 1, dtype=torch.int32, device=gpu)
    indptr[1::2] = pages
    indptr[S] = 1
    last = torch.full((S,), P, dtype=torch.int32, device=gpu)
    q = torch.randn((S, D), generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    need = lib.vtx_quant_decode_attention_workspace_len(S, 1, 1, D, P, 0, 0, pages)
    assert need > 0
    room = 1 << 20
    ws = torch.full((need + 2 * room,), 7.0, device=gpu)
    out = torch.full((S * D + 2 * room,), 7.0, dtype=torch.bfloat16, device=gpu)
    stream = torch.cuda.current_stream().cuda_stream
    rc = lib.vtx_quant_decode_attention(
        q.data_ptr(), (ctypes.c_int64 * 3)(D, D, D), out[room:].data_ptr(), kc.data_ptr(), vc.data_ptr(),
        sc.data_ptr(), 1, indptr.data_ptr(), indices.data_ptr(), pages, last.data_ptr(), S, 1, 1, D, P, 0,
        _hip.CODES_INT8, D ** -0.5, 0.0, 0, None, 0, ws[room:].data_ptr(), need, stream)
    assert rc == 0
    torch.cuda.synchronize()
    for t in (ws, out):
        assert bool((t[:room] == 7).all()) and bool((t[-room:] == 7).all())
    assert int(out[room:-room].view(S, D)[1:-1:2].count_nonzero()) == 0  # segments without pages


def test_reductions_refuse_heads_whose_tiles_pass_an_int():
    """256 pages of a block times the heads, and a round of the workgroups more."""
    lib, p = _hip.load_library(), [0x10000 * (i + 1) for i in range(4)]
    for heads in ((1 << 31) // 256 - 1, (1 << 31) // 256 - 4):
        assert lib.vtx_page_reduce_quant(p[0], p[1], 1 << 31, 1, 1, _hip.CODES_INT8, 1, (ctypes.c_void_p * 1)(p[2]),
                                         (ctypes.c_int32 * 1)(0), (ctypes.c_int32 * 1)(_hip.REDUCE_MEAN), 1 << 31, p[3],
                                         256, heads, None) == -1
        assert b"too many heads" in lib.vtx_last_error()


# --------------------------------------------------- rows that are no numbers
@pytest.mark.gpu
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("H,P,D,pages", [(2, 16, 128, 9), (2, 16, 64, 9), (1, 64, 256, 5), (2, 33, 512, 5),
                                         (3, 5, 128, 9), (2, 16, 80, 9), (1, 7, 3, 9), (8, 16, 128, 700),
                                         (8, 16, 64, 2100)])
def test_page_reductions_of_rows_that_are_no_numbers(gpu, H, P, D, pages, codes):
    """Every statistic of a page with such a row is NaN, the extremes among them,
    and of every other page what it was; a NaN code is one of its column."""
    gen = torch.Generator().manual_seed(D)
    kc, vc, sc = _random_pool(pages * H, P, D, codes, gen, gpu)
    loc = torch.arange(pages * P, device=gpu)
    types = [_hip.REDUCE_MEAN, _hip.REDUCE_MAX, _hip.REDUCE_MIN, _hip.REDUCE_L2NORM]

    def reduce(kinds):
        outs = [torch.zeros((pages * H, 1, D), dtype=torch.bfloat16, device=gpu) for _ in kinds]
        _hip.page_reduce_quant(kc, sc, False, outs, kinds, loc, H, P, 1)
        return outs

    sets = [[t] for t in types] + [[_hip.REDUCE_MAX, _hip.REDUCE_MIN], types]
    before = [reduce(kinds) for kinds in sets]
    x = torch.randn((3, H, D), generator=gen).to(gpu)
    x[0, 0, 0], x[1, H - 1, D - 1], x[2, 0, D // 2] = math.inf, math.nan, -math.inf
    # the first, a middle and the last token of three pages
    set_kv_buffer_quant(kc, vc, sc, x, x, torch.tensor([0, P + P // 2, 3 * P - 1], device=gpu), P)
    bad = torch.zeros((pages * H, 1, D), dtype=torch.bool, device=gpu)
    bad[[0, 2 * H - 1, 2 * H]] = True
    if codes == E4M3:
        kc.view(torch.uint8)[4 * H, P // 3, 1] = 0x7F
        bad[4 * H, 0, 1] = True
    keep = torch.ones(pages * H, dtype=torch.bool, device=gpu)
    keep[:3 * H], keep[4 * H] = False, codes != E4M3
    for kinds, old in zip(sets, before):
        for got, was in zip(reduce(kinds), old):
            assert torch.equal(got.isnan(), bad), kinds
            assert torch.equal(got[keep], was[keep])


# ------------------------------------------------------------- known bounds
@pytest.mark.parametrize("segments,D,window,most", [
    (256, 64, 0, 2048), (256, 128, 0, 2048), (256, 256, 0, 1024), (512, 128, 0, 2048), (2048, 64, 0, 2048),
    (512, 128, 1, 2048), (512, 256, 1, 1024), (1024, 128, 1, 4096), (2048, 256, 1, 4096), (8, 128, 0, 512),
    (8, 128, 1, 1024), (8, 256, 1, 768)])
def test_known_bounds_up_to_which_every_segment_has_a_workgroup(segments, D, window, most):
    """Past them the table is looked at, which needs the workspace: ragged batches of
    longer requests are slower with a workgroup each."""
    need = _hip.load_library().vtx_quant_decode_attention_workspace_len
    for tokens, divided in ((most, False), (most + 1, True)):
        asked = (tokens, 0) if window else (0, tokens)
        assert (need(segments, 1, 2, D, 16, *asked, 1 << 20) > 0) == divided
