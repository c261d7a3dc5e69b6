"""set_kv_buffer_rope: rotation of queries and keys on the way into the paged
pools, against the formula in 64 bits, and its refusals."""
import ctypes

import pytest
import torch

from vortex_torch import _hip
from vortex_torch.cache import set_kv_buffer_rope

SENTINEL = 7.0
PAGE_SPARE = 3


def _table(rows, rotary, device="cpu"):
    half = rotary // 2
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def _rotated(x, table, positions, interleaved):
    """(the rotated rows, what the fp32 steps may be off) in 64 bits, on x's device."""
    R = table.shape[1]
    y, cs = x.double().clone(), table[positions].double()[:, None]
    c, s = cs[..., :R // 2], cs[..., R // 2:]
    at = [slice(0, R, 2), slice(1, R, 2)] if interleaved else [slice(0, R // 2), slice(R // 2, R)]
    a, b = x.double()[..., at[0]], x.double()[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    # one product rounded, then one fused step: 2^-24 of the product and 2^-24 of the sum, each at most |a| + |b|
    off = torch.zeros_like(y)
    off[..., at[0]] = off[..., at[1]] = 2.0 ** -23 * (a.abs() + b.abs())
    return y, off


def _close(got, want, off, dtype):
    half_step = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * half_step  # half a step among the smallest values
    bound = off + half_step * (want.abs() + off) + least
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


def _tensors(n, heads, D, dtype, layout, gen, device):
    """q, k and v [n, h, D] in one of several layouts."""
    randn = lambda *s: torch.randn(s, generator=gen).to(dtype).to(device)  # noqa: E731
    if layout == "fused":
        return [t.unflatten(1, (-1, D)) for t in randn(n, sum(heads) * D).split([h * D for h in heads], dim=1)]
    if layout == "heads_first":
        return [randn(h, n, D).transpose(0, 1) for h in heads]
    if layout == "odd":  # rows that begin one element past an aligned address
        return [randn(n, h, D + 1)[..., 1:] for h in heads]
    return [randn(n, h, D) for h in heads]


def _slots(n, pages, P, gen):
    return torch.randperm(pages * P, generator=gen)[:n]


def _check(n, Hq, H, D, R, P, dtype, layout, interleaved, device, in_place=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = _tensors(n, (Hq, H, H), D, dtype, layout, gen, device)
    pages, rows = (n + P - 1) // P + PAGE_SPARE, 4096
    loc, positions = _slots(n, pages, P, gen).to(device), torch.randint(0, rows, (n,), generator=gen).to(device)
    if n > 4:  # padding, slots and positions out of range
        loc[n - 1], loc[1] = -1, pages * P + 3
        positions[2], positions[3] = -1, rows
    table = _table(rows, R, device)
    kc = torch.full((pages * H, P, D), SENTINEL, dtype=dtype, device=device)
    vc = kc.clone()
    wants = [_rotated(t, table, positions.clamp(0, rows - 1), interleaved) for t in (q, k)]
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    out = q if in_place else torch.full((n, Hq, D), SENTINEL, dtype=dtype, device=device)
    got = set_kv_buffer_rope(kc, vc, q, k, v, loc, P, positions, table, interleaved=interleaved, q_out=out)
    assert got is out
    placed = (positions >= 0) & (positions < rows)
    stored = placed & (loc >= 0) & (loc < pages * P)
    _close(got[placed], wants[0][0][placed], wants[0][1][placed], dtype)
    assert torch.equal(got[~placed], q0[~placed] if in_place else torch.full_like(got[~placed], SENTINEL))
    at = loc[stored]
    k4, v4 = kc.view(pages, H, P, D), vc.view(pages, H, P, D)
    _close(k4[at // P, :, at % P], wants[1][0][stored], wants[1][1][stored], dtype)
    assert torch.equal(v4[at // P, :, at % P], v0[stored])
    k4[at // P, :, at % P] = SENTINEL
    v4[at // P, :, at % P] = SENTINEL
    assert bool((kc == SENTINEL).all()) and bool((vc == SENTINEL).all())  # all other rows as they were
    assert torch.equal(k, k0) and torch.equal(v, v0) and (in_place or torch.equal(q, q0))


SHAPES = [  # tokens, query heads, kv heads, head_dim, rotary_dim, page
    (1, 1, 1, 2, 2, 1), (5, 3, 2, 7, 6, 16), (6, 4, 2, 64, 64, 16), (9, 16, 8, 128, 128, 16), (33, 2, 1, 80, 80, 8),
    (70, 8, 2, 128, 64, 32), (7, 6, 3, 256, 96, 5), (257, 1, 1, 64, 16, 64), (40, 5, 5, 96, 48, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rope_append(gpu, shape, dtype, interleaved):
    for layout in ("fused", "apart", "heads_first", "odd"):
        _check(*shape, dtype, layout, interleaved, gpu, seed=shape[0])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["fused", "apart", "odd"])
def test_rope_append_in_place(gpu, layout):
    _check(37, 16, 8, 128, 128, 16, torch.bfloat16, layout, False, gpu, in_place=True)
    _check(37, 4, 2, 80, 40, 16, torch.float16, layout, True, gpu, in_place=True)


@pytest.mark.gpu
def test_rope_append_large_prefill_and_no_queries(gpu):
    _check(5000, 8, 2, 128, 128, 16, torch.bfloat16, "fused", False, gpu)
    gen = torch.Generator().manual_seed(1)
    _, k, v = _tensors(21, (2, 2, 2), 64, torch.bfloat16, "fused", gen, gpu)
    kc, vc = torch.zeros((2, 8 * 2, 16, 64), dtype=torch.bfloat16, device=gpu)
    loc, positions, table = torch.arange(21, device=gpu), torch.arange(21, device=gpu), _table(64, 64, gpu)
    assert set_kv_buffer_rope(kc, vc, None, k, v, loc, 16, positions, table) is None
    want, off = _rotated(k, table, positions, False)
    _close(kc.view(8, 2, 16, 64)[loc // 16, :, loc % 16], want, off, torch.bfloat16)
    empty = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=gpu)
    assert set_kv_buffer_rope(kc, vc, empty, empty, empty, loc[:0], 16, positions[:0], table).shape == (0, 2, 64)


@pytest.mark.gpu
def test_rope_append_agrees_with_plain_store_bit_for_bit(gpu):
    """Position 0 turns nothing: the pools are set_kv_buffer's."""
    from vortex_torch.cache import set_kv_buffer_launcher

    gen = torch.Generator().manual_seed(2)
    q, k, v = _tensors(50, (4, 2, 2), 128, torch.bfloat16, "apart", gen, gpu)
    loc = _slots(50, 6, 16, gen).to(gpu)
    pools = torch.zeros((4, 12, 16, 128), dtype=torch.bfloat16, device=gpu)
    got = set_kv_buffer_rope(pools[0], pools[1], q, k, v, loc, 16, torch.zeros_like(loc), _table(8, 128, gpu))
    set_kv_buffer_launcher(pools[2], pools[3], k, v, loc, 16)
    assert torch.equal(pools[:2], pools[2:]) and torch.equal(got, q)


@pytest.mark.gpu
def test_rope_append_into_layout_tagged_pools_and_after_a_carried_mean(gpu):
    """A flow's pools (vTensors), with the page-finish mean that forward_cache
    left for the next launch: it sees the pool as it was before the call."""
    import workloads as W
    from vortex_torch import flow as vflow
    from vortex_torch.abs import FORMAT, as_vtensor

    batch = W.c1()
    H, G, D, P = batch.num_kv_heads, batch.group_size, batch.head_dim, batch.page_size
    ictx, cctx = W.make_contexts(batch, gpu)
    flow = vflow.build_vflow("block_sparse_attention")
    k = W.k_pool(batch, 10, gpu)
    centroids = torch.zeros((batch.pool_pages * H, 1, D), device=gpu, dtype=torch.bfloat16)
    cache = {"k": as_vtensor(k, FORMAT.PAGED), "v": as_vtensor(torch.zeros_like(k), FORMAT.PAGED),
             "centroids": as_vtensor(centroids, FORMAT.PAGED)}
    loc = torch.tensor([5 * P + P - 1], device=gpu)
    for c in (ictx, cctx):
        c.profile()
    flow.forward_cache(cache, loc, cctx)
    for c in (ictx, cctx):
        c.execute()
    before = k.view(-1, H, P, D)[5].float().mean(1)
    flow.forward_cache(cache, loc, cctx)
    gen = torch.Generator().manual_seed(4)
    q, nk, nv = _tensors(1, (H * G, H, H), D, torch.bfloat16, "fused", gen, gpu)
    table = _table(64, D, gpu)
    set_kv_buffer_rope(cache["k"], cache["v"], q, nk, nv, loc, P, torch.tensor([9], device=gpu), table)
    got = centroids.view(-1, H, D)[5].float()
    assert bool(((got - before).abs() <= 2.0 ** -8 * before.abs() + 2.0 ** -20).all())
    want, off = _rotated(nk, table, torch.tensor([9], device=gpu), False)
    _close(k.view(-1, H, P, D)[5, :, P - 1], want[0], off[0], torch.bfloat16)


@pytest.mark.gpu
def test_rope_append_offsets_past_32_bits(gpu):
    """The last page of pools of over 2^32 bytes, the last row of a table as large."""
    D, P, pages = 128, 16, (1 << 32) // (16 * 128 * 2) + 9
    rows = (1 << 32) // (4 * D) + 5
    kc, vc = (torch.zeros((pages, P, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    table = torch.zeros((rows, D), device=gpu)
    table[-1] = _table(1000, D, gpu)[-1]
    k = torch.randn((1, 1, D), dtype=torch.bfloat16, device=gpu)
    loc, positions = (torch.tensor([x], device=gpu) for x in (pages * P - 1, rows - 1))
    q = set_kv_buffer_rope(kc, vc, k, k, k, loc, P, positions, table)
    want, off = _rotated(k, table, positions, False)
    _close(q, want, off, torch.bfloat16)
    assert torch.equal(kc[-1, -1], q[0, 0]) and torch.equal(vc[-1, -1], k[0, 0])
    assert int(kc[:64].count_nonzero()) == 0 and int(kc[-64:].count_nonzero()) <= D


@pytest.mark.gpu
@pytest.mark.parametrize("H,P,D", [(1, 16, 128), (2, 16, 64), (3, 5, 7), (4, 16, 128), (8, 16, 128), (8, 1, 64)])
def test_rope_append_slots_far_past_the_pool(gpu, H, P, D):
    """A slot outside the pool stores nothing however large it is: a row of
    heads x slot leaves 64 bits from 2^63 / H on.  Guards lie on both sides."""
    pages, guard = 7, 130 * H * P
    far = [pages * P, (1 << 31) - 1, 1 << 31, 1 << 32, 1 << 40, (1 << 63) // H - 1, (1 << 63) - 1, (1 << 63) - P,
           *(1 << b for b in range(57, 63)), *((1 << b) + 3 * P + 2 for b in range(57, 63)), -1, -(1 << 63)]
    loc = torch.tensor([pages * P - 1, *(min(x, (1 << 63) - 1) for x in far)], device=gpu)
    n = loc.numel()
    buffers = torch.full((2, guard + pages * H * P + guard, D), SENTINEL, dtype=torch.bfloat16, device=gpu)
    kc, vc = (b[guard:-guard].view(pages * H, P, D) for b in buffers)
    q, k, v = _tensors(n, (H, H, H), D, torch.bfloat16, "apart", torch.Generator().manual_seed(6), gpu)
    table, positions = _table(64, D // 2 * 2, gpu), torch.arange(n, device=gpu)
    got = set_kv_buffer_rope(kc, vc, q, k, v, loc, P, positions, table)
    _close(got, *_rotated(q, table, positions, False), torch.bfloat16)  # (queries are rotated all the same)
    want, off = _rotated(k, table, positions, False)
    _close(kc.view(pages, H, P, D)[-1, :, -1], want[0], off[0], torch.bfloat16)
    assert torch.equal(vc.view(pages, H, P, D)[-1, :, -1], v[0])
    kc.view(pages, H, P, D)[-1, :, -1] = SENTINEL
    vc.view(pages, H, P, D)[-1, :, -1] = SENTINEL
    assert bool((buffers == SENTINEL).all())


@pytest.mark.gpu
def test_rope_append_streams_and_graphs(gpu):
    gen = torch.Generator().manual_seed(3)
    q, k, v = _tensors(24, (4, 2, 2), 128, torch.bfloat16, "fused", gen, gpu)
    loc, positions = _slots(24, 4, 16, gen).to(gpu), torch.arange(24, device=gpu)
    table = _table(512, 128, gpu)
    kc, vc = torch.zeros((2, 8, 16, 128), dtype=torch.bfloat16, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = set_kv_buffer_rope(kc, vc, q, k, v, loc, 16, positions, table)
    torch.cuda.synchronize()
    out = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        set_kv_buffer_rope(kc, vc, q, k, v, loc, 16, positions, table, q_out=out)
    for step in range(3):
        positions += 31
        kc.zero_()
        graph.replay()
        eager_k, eager_v = torch.zeros_like(kc), torch.zeros_like(vc)
        eager = set_kv_buffer_rope(eager_k, eager_v, q, k, v, loc, 16, positions, table)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(kc, eager_k) and torch.equal(vc, eager_v)


# ------------------------------------------------------------- refusals (CPU)
def _arguments(**changes):
    n, Hq, H, D, P = 3, 4, 2, 16, 8
    bf = dict(dtype=torch.bfloat16)
    a = dict(k_cache=torch.zeros((2 * H, P, D), **bf), v_cache=torch.zeros((2 * H, P, D), **bf),
             q=torch.zeros((n, Hq, D), **bf), new_k=torch.zeros((n, H, D), **bf), new_v=torch.zeros((n, H, D), **bf),
             loc=torch.arange(n), page_size=P, positions=torch.arange(n), cos_sin_cache=torch.zeros((10, D)))
    a.update(changes)
    return a


_POOL = torch.zeros((4, 8, 16), dtype=torch.bfloat16)
_ARENA = torch.zeros(1024, dtype=torch.bfloat16)
_ROWS = torch.zeros((3, 8 * 16), dtype=torch.bfloat16).unflatten(1, (8, 16))


@pytest.mark.parametrize("changes, says", [
    (dict(loc=torch.arange(3, dtype=torch.int32)), "loc must be torch.int64"),
    (dict(positions=torch.arange(3, dtype=torch.int32)), "positions must be torch.int64"),
    (dict(cos_sin_cache=torch.zeros((10, 16), dtype=torch.float64)), "cos_sin_cache must be torch.float32"),
    (dict(cos_sin_cache=torch.zeros((10, 32))[:, ::2]), "cos_sin_cache must be contiguous"),
    (dict(cos_sin_cache=torch.zeros(160)), "cos_sin_cache must be \\[positions"),
    (dict(new_v=torch.zeros((3, 1, 16), dtype=torch.bfloat16)), "must both be"),
    (dict(q=torch.zeros((3, 4, 8), dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros((2, 4, 16), dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros((3, 4, 16))), "q is torch.float32"),
    (dict(q=torch.zeros((3, 4, 32), dtype=torch.bfloat16)[..., ::2]), "q must have dense rows"),
    (dict(k_cache=torch.zeros((4, 8, 16))), "k_cache is torch.float32"),
    (dict(v_cache=torch.zeros((4, 8, 32), dtype=torch.bfloat16)[..., :16]), "must be contiguous"),
    (dict(v_cache=torch.zeros((6, 8, 16), dtype=torch.bfloat16)), "must be \\[pages"),
    (dict(page_size=16), "must be \\[pages"),
    (dict(k_cache=torch.zeros((3, 8, 16), dtype=torch.bfloat16), v_cache=torch.zeros((3, 8, 16), dtype=torch.bfloat16)),
     "not pages of 2"),
    (dict(loc=torch.arange(2)), "shorter"),
    (dict(positions=torch.arange(2)), "shorter"),
    (dict(k_cache=_POOL, v_cache=_POOL), "share memory"),
    (dict(k_cache=_POOL, new_k=_POOL.view(-1)[:96].view(3, 2, 16)), "new_k lies in the pools"),
    (dict(q=None, q_out=torch.zeros((3, 4, 16), dtype=torch.bfloat16)), "q_out without q"),
    (dict(q_out=torch.zeros((3, 2, 16), dtype=torch.bfloat16)), "q_out must be"),
    (dict(q_out=torch.zeros((1, 4, 16), dtype=torch.bfloat16).expand(3, 4, 16)), "q_out has rows"),
    (dict(q=_ROWS[:, :4], q_out=_ROWS[:, 1:5]), "q_out shares memory with q"),
    (dict(q=_ROWS[:, :4], q_out=_ROWS[:, :4], new_k=_ROWS[:, 3:5]), "q_out shares memory with new_k"),
    (dict(new_k=torch.zeros((3, 2, 16), dtype=torch.float64), ), "must be bfloat16, float16 or float32"),
])
def test_rope_append_refusals(monkeypatch, changes, says):
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_current_device", lambda: 0)
    with pytest.raises(RuntimeError, match=says):
        set_kv_buffer_rope(**_arguments(**changes))


@pytest.mark.parametrize("changes, says", [
    (dict(k_cache=_ARENA[256:768].view(4, 8, 16), new_k=_ARENA[192:288].view(3, 2, 16)), "new_k lies in the pools"),
    (dict(v_cache=_ARENA[256:768].view(4, 8, 16), new_v=_ARENA[161:257].view(3, 2, 16)), "new_v lies in the pools"),
    (dict(k_cache=_ARENA[256:768].view(4, 8, 16), q=_ARENA[:192].view(3, 4, 16).as_strided((3, 4, 16), (128, 16, 1))),
     "q lies in the pools"),
    (dict(k_cache=_ARENA[256:768].view(4, 8, 16), q_out=_ARENA[65:257].view(3, 4, 16)), "q_out lies in the pools"),
])
def test_rope_append_refuses_rows_that_reach_into_a_pool(monkeypatch, changes, says):
    """They begin before it."""
    test_rope_append_refusals(monkeypatch, changes, says)


def test_rope_append_takes_rows_that_end_where_a_pool_begins(monkeypatch):
    """Rows up to a pool's first byte, and from its last one on, are answered."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    monkeypatch.setattr(_hip, "_lib", Lib())
    monkeypatch.setattr(_hip, "_device_index", lambda *t: 0)
    monkeypatch.setattr(_hip, "_current_device", lambda: 0)
    monkeypatch.setattr(_hip, "_stream_of", lambda index: 0)
    pool = _ARENA[256:768].view(4, 8, 16)
    for at in (0, 64, 768, 800):  # (192 elements of q, 96 of new_k and of new_v)
        q, rows = _ARENA[at:at + 192].view(3, 4, 16), _ARENA[at:at + 96].view(3, 2, 16)
        for changes in (dict(q=q), dict(new_k=rows), dict(new_v=rows), dict(q_out=q)):
            set_kv_buffer_rope(**_arguments(k_cache=pool, **changes))
            set_kv_buffer_rope(**_arguments(v_cache=pool, **changes))
    assert calls == ["vtx_set_kv_buffer_rope"] * 32


def test_rope_append_needs_a_gpu():
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        set_kv_buffer_rope(**_arguments())


def test_slices_of_one_projection_do_not_overlap():
    q, k, v = torch.zeros((5, 8 * 16)).split([64, 32, 32], dim=1)
    q, k, v = (t.unflatten(1, (-1, 16)) for t in (q, k, v))
    for a in (q, k, v):
        assert _hip._rows_distinct(a)
        for b in (q, k, v):
            assert _hip._tokens_apart(a, b) == (a is not b)
    t = torch.zeros((4, 5, 16)).transpose(0, 1)
    assert _hip._rows_distinct(t) and not _hip._rows_distinct(torch.zeros((1, 4, 16)).expand(5, 4, 16))
    assert not _hip._rows_distinct(torch.zeros(100).as_strided((5, 4, 16), (8, 16, 1)))


def test_rope_append_c_refusals():
    lib = _hip.load_library()
    strides = (ctypes.c_int64 * 8)(64, 16, 64, 16, 32, 16, 32, 16)
    p = [0x10000 * (i + 1) for i in range(9)]

    def call(nnz=3, heads=2, dim=16, rotary=16, dtype=0, page=8, q=p[0], loc=p[4]):
        return lib.vtx_set_kv_buffer_rope(p[5], p[6], 32, q, p[1], p[2], p[3], strides, loc, p[7], p[8], 10, nnz, 4,
                                          heads, dim, rotary, dtype, page, 0, None)

    for kw, says in ((dict(nnz=-1), b"bad sizes"), (dict(heads=0), b"bad sizes"), (dict(page=0), b"bad sizes"),
                     (dict(rotary=3), b"rotary_dim"), (dict(rotary=18), b"rotary_dim"), (dict(rotary=0), b"rotary_dim"),
                     (dict(dtype=3), b"element type"), (dict(q=None), b"null"), (dict(loc=None), b"null"),
                     (dict(heads=1 << 30, dim=1 << 20), b"too wide")):
        assert call(**kw) == -1 and says in lib.vtx_last_error(), (kw, lib.vtx_last_error())
    assert call(nnz=0) == 0
