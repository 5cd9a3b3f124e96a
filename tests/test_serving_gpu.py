"""Attention of packed sequences, a key / value cache in pages and attention
over it, against their formulas in 64 bits."""
import numpy as np
import pytest

from fusilli_amd import capi
from helpers import HT
from serving import (HALF_STEP, Cache, attend, check, cpp_binary, rotation_table, starts, to_groups, turn,
                     turn_bound)

pytestmark = pytest.mark.gpu
SENTINEL = 77.0  # (exact in every type)


def rows_strides(dims, how):
    t, h, d = dims
    return {"dense": [h * d, d, 1], "heads": [d, t * d, 1], "wide": [h * d + 64, d, 1], "fused": [3 * h * d, d, 1]}[how]


def rows_of(rng, dims, dtype, how="dense", std=1.0):
    return HT.from_logical(rng.standard_normal(dims) * std, dtype, rows_strides(dims, how))


def ints(ctx, values):
    return ctx.to_device(np.asarray(values, np.int32))


# ---- packed ------------------------------------------------------------------
def run_packed(ctx, q, k, v, offsets, causal, kv_offsets=None, scale=None, o_how="dense"):
    dims = [q.dims[0], q.dims[1], v.dims[2]]
    o = HT.from_logical(np.full(dims, SENTINEL), q.dtype, rows_strides(dims, o_how))
    d = capi.SdpaPackedDesc()
    d.q, d.k, d.v, d.o = q.desc(), k.desc(), v.desc(), o.desc()
    d.batch, d.is_causal, d.has_kv_offsets = len(offsets) - 1, int(causal), int(kv_offsets is not None)
    if scale is not None:
        d.has_scale, d.scale = 1, scale
    bufs = [t.upload(ctx) for t in (q, k, v, o)]
    at = ints(ctx, offsets), None if kv_offsets is None else ints(ctx, kv_offsets)
    ctx.sdpa_packed_fwd(d, *bufs[:3], at[0], bufs[3], kv_offsets=at[1])
    return o.fetch(ctx, bufs[3]).logical(), ctx.lib.fhip_sdpa_packed_fwd_supported(d)


def check_packed(q, k, v, offsets, causal, got, kv_offsets=None, scale=None, what=""):
    kv = offsets if kv_offsets is None else kv_offsets
    outside = np.ones(q.dims[0], bool)
    ql, kl, vl = (t.logical().astype(np.float64) for t in (q, k, v))
    for b in range(len(offsets) - 1):
        r, s = slice(offsets[b], offsets[b + 1]), slice(kv[b], kv[b + 1])
        n, m = offsets[b + 1] - offsets[b], kv[b + 1] - kv[b]
        outside[r] = False
        if n == 0:
            continue
        seen = np.clip(m - n + 1 + np.arange(n), 0, m) if causal else np.full(n, m)
        ref, far = attend(ql[r], kl[s], vl[s], seen, q.dtype, scale)
        check(got[r], ref, far, f"{what} sequence {b}")
    assert (got[outside] == SENTINEL).all(), "rows of no sequence were written"


PACKED = [
    # lengths, query heads, key heads, causal
    ([1], 1, 1, True),
    ([1, 1, 1], 4, 4, True),
    ([0, 5, 0, 0, 17, 1, 0], 4, 2, True),
    ([63, 64, 65], 2, 1, True),
    ([300], 3, 1, True),              # 900 grouped rows
    ([257, 2, 513, 31], 8, 2, True),
    ([31, 130, 1], 7, 1, True),       # rows of a position cross tiles
    ([700, 20], 2, 2, True),
    ([5, 100, 64], 4, 2, False),
    ([190, 333, 1], 6, 2, False),
    ([16] * 70, 2, 1, True),          # more sequences than a wavefront has lanes
]


@pytest.mark.parametrize("lens,hq,hkv,causal", PACKED)
@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.HALF])
@pytest.mark.parametrize("d", [64, 128])
def test_packed(ctx, lens, hq, hkv, causal, dtype, d):
    rng = np.random.default_rng([1, sum(lens), hq, d])
    t = sum(lens)
    q, k, v = rows_of(rng, [t, hq, d], dtype, std=2.0), rows_of(rng, [t, hkv, d], dtype), rows_of(rng, [t, hkv, d], dtype)
    at = starts(lens)
    got, _ = run_packed(ctx, q, k, v, at, causal)
    check_packed(q, k, v, at, causal, got)


@pytest.mark.parametrize("dtype,d,dv", [(capi.FLOAT, 64, 64), (capi.FLOAT, 33, 50), (capi.BFLOAT16, 80, 80), (capi.HALF, 96, 128),
                                        (capi.HALF, 1, 1), (capi.BFLOAT16, 256, 512)])
def test_packed_other_sizes_and_types(ctx, dtype, d, dv):
    rng = np.random.default_rng([2, d, dv])
    lens = [3, 0, 70, 1]
    q, k, v = rows_of(rng, [74, 4, d], dtype), rows_of(rng, [74, 2, d], dtype), rows_of(rng, [74, 2, dv], dtype)
    got, level = run_packed(ctx, q, k, v, starts(lens), True)
    assert level == 1
    check_packed(q, k, v, starts(lens), True, got)


@pytest.mark.parametrize("how", ["heads", "wide", "fused"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_strides_scale_and_rows_of_no_sequence(ctx, how, d, causal):
    rng = np.random.default_rng([3, d])
    at = np.array([2, 2, 90, 200, 207], np.int32)  # rows 0, 1 and 207 .. 209 belong to none
    q, k, v = (rows_of(rng, [210, h, d], capi.BFLOAT16, how) for h in (6, 2, 2))
    got, _ = run_packed(ctx, q, k, v, at, causal, scale=0.31, o_how=how)
    check_packed(q, k, v, at, causal, got, scale=0.31)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_packed_behind_a_prefix(ctx, d, causal, scale):
    # as many keys as rows, more, fewer (rows that see none), none
    rng = np.random.default_rng([4, d])
    lens, keys = [7, 100, 40, 9, 0, 1, 70], [7, 400, 25, 0, 12, 333, 70]
    q = rows_of(rng, [sum(lens), 4, d], capi.HALF)
    k, v = (rows_of(rng, [sum(keys), 2, d], capi.HALF) for _ in range(2))
    got, _ = run_packed(ctx, q, k, v, starts(lens), causal, kv_offsets=starts(keys), scale=scale)
    check_packed(q, k, v, starts(lens), causal, got, kv_offsets=starts(keys), scale=scale)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_neighbours_stay_apart(ctx, d):
    # the other sequences' keys and values are infinite or NaN; so are a sequence's own later ones
    rng = np.random.default_rng([5, d])
    lens = [40, 300, 23]
    at = starts(lens)
    q, k, v = (rng.standard_normal([363, h, d]) for h in (4, 2, 2))
    k[:40], v[:40], k[340:], v[340:] = np.nan, np.inf, -np.inf, np.nan
    q, k, v = (HT.from_logical(x, capi.BFLOAT16) for x in (q, k, v))
    got, _ = run_packed(ctx, q, k, v, at, True)
    ref, far = attend(*(t.logical().astype(np.float64)[40:340] for t in (q, k, v)), np.arange(300) + 1, capi.BFLOAT16)
    check(got[40:340], ref, far)
    v = v.logical()
    v[339] = np.inf  # only the last row sees it, and rows whose 64 keys hold it
    got, _ = run_packed(ctx, q, k, HT.from_logical(v, capi.BFLOAT16), at, True)
    check(got[40:296], ref[:256], far[:256])
    assert not np.isfinite(got[339]).any()


@pytest.mark.parametrize("d", [64, 128])
def test_packed_high_scores_move_the_reference_point(ctx, d):
    # scores that rise by hundreds along the keys, and fall again
    rng = np.random.default_rng([6, d])
    n = 520
    q = np.ones([n, 2, d]) + 0.01 * rng.standard_normal([n, 2, d])
    ramp = 40 * np.sin(np.arange(n) / 90)[:, None, None]
    k = ramp + rng.standard_normal([n, 1, d])
    q, k, v = (HT.from_logical(x, capi.HALF) for x in (q, k, rng.standard_normal([n, 1, d])))
    got, _ = run_packed(ctx, q, k, v, starts([n]), True)
    check_packed(q, k, v, starts([n]), True, got)


# ---- append and read -----------------------------------------------------------
def run_append(ctx, cache, lengths, offsets, k, v, q=None, table=None, positions=None, interleaved=False,
               k_out=True, in_place=False):
    d = capi.CacheAppendDesc()
    d.k, d.v, d.cache, d.interleaved = k.desc(), v.desc(), cache.desc(), int(interleaved)
    outs = {}
    kw = {}
    at = cache.upload(ctx, lengths)
    bufs = {"k": k.upload(ctx), "v": v.upload(ctx)}
    if q is not None:
        bufs["q"] = q.upload(ctx)
        qo = q if in_place else HT.from_logical(np.full(q.dims, SENTINEL), q.dtype)
        d.q, d.q_out = q.desc(), qo.desc()
        kw["q"], kw["q_out"] = bufs["q"], bufs["q"] if in_place else qo.upload(ctx)
        outs["q"] = qo
    if k_out:
        ko = k if in_place else HT.from_logical(np.full(k.dims, SENTINEL), k.dtype)
        d.k_out = ko.desc()
        kw["k_out"] = bufs["k"] if in_place else ko.upload(ctx)
        outs["k"] = ko
    if table is not None:
        d.rotation = capi.TensorDesc.make(table.shape, [table.shape[1], 1], capi.FLOAT)
        kw["rotation"] = ctx.to_device(table)
    if positions is not None:
        d.has_positions = 1
        kw["positions"] = ints(ctx, positions)
    ctx.cache_append(d, at, bufs["k"], bufs["v"], ints(ctx, offsets), **kw)
    cache.fetch(ctx)
    if "q" in outs:
        outs["q"].fetch(ctx, kw["q_out"])
    if "k" in outs:
        outs["k"].fetch(ctx, kw["k_out"])
    return {n: t.logical() for n, t in outs.items()}, ctx.lib.fhip_cache_append_supported(d)


def one_step(x, dtype):
    """A step of the type at x (below the smallest normal: of the smallest)."""
    low = {capi.BFLOAT16: -126, capi.HALF: -14, capi.FLOAT: -126}[dtype]
    return 2 * HALF_STEP[dtype] * 2.0 ** np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-300))), low)


def check_turned(got, x, table, pos, interleaved, dtype):
    """q_out / k_out: half a step, and what three roundings in f32 move it by."""
    ref = turn(x, table, pos, interleaved)
    far = turn_bound(x, table, pos, interleaved, dtype)
    check(got, ref, far + 0.5 * one_step(np.abs(ref) + far, dtype) * (1 + 1e-9))


def check_held(cache, before, after, where, x, group, dtype, what):
    """A pool `after` an append: the rows x at `where` ((pages, slots)), all else as `before`."""
    page, slot = where
    expect = [t.copy() for t in before]
    if not group:
        expect[0][page, :, slot] = x
    else:
        code, scale, low = to_groups(x, group)
        expect[0][page, :, slot] = code[..., ::2] | code[..., 1::2] << 4
        expect[1][page, :, slot] = np.stack([scale, low], -1).reshape(*scale.shape[:-1], -1)
    for a, e in zip(after, expect):
        assert np.array_equal(a, e, equal_nan=True), f"{what}: {(a != e).sum()} differ"


APPEND = [
    # rows per sequence, keys they follow, page size
    ([1], [0], 16),
    ([1, 1, 1], [0, 15, 16], 16),
    ([0, 9, 0, 33, 1], [4, 7, 0, 31, 64], 32),
    ([70, 5], [0, 100], 64),
    ([20, 3], [13, 2], 5),
    ([3, 1], [0, 0], 1),
]


@pytest.mark.parametrize("lens,past,page", APPEND)
@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.HALF, capi.FLOAT])
@pytest.mark.parametrize("d,rotary,interleaved,group", [
    (128, 128, False, 0), (128, 128, False, 64), (128, 64, True, 32), (64, 64, True, 64), (64, 32, False, 32),
    (128, 48, False, 128), (80, 80, False, 0), (80, 20, True, 16), (50, 10, False, 10), (64, 0, False, 0)])
def test_append(ctx, lens, past, page, dtype, d, rotary, interleaved, group):
    rng = np.random.default_rng([7, sum(lens), d, rotary, group])
    t, keys = sum(lens), [n + p for n, p in zip(lens, past)]
    cache = Cache(rng, keys, 2, d, page, dtype, group)
    q, k, v = rows_of(rng, [t, 6, d], dtype), rows_of(rng, [t, 2, d], dtype, "wide"), rows_of(rng, [t, 2, d], dtype, "fused")
    before = [[p.logical() for p in x] for x in (cache.k, cache.v)]
    x = {n: r.logical().astype(np.float64) for n, r in (("q", q), ("k", k), ("v", v))}
    table = rotation_table(max(keys) + 1, rotary) if rotary else None
    got, _ = run_append(ctx, cache, keys, starts(lens), k, v, q, table, interleaved=interleaved)
    seq = np.repeat(np.arange(len(lens)), lens)
    place = np.concatenate([np.arange(p, p + n) for n, p in zip(lens, past)])
    for n in ("q", "k"):
        if rotary:
            check_turned(got[n], x[n], table, place, interleaved, dtype)
        else:
            assert np.array_equal(got[n], x[n])
    where = cache.table[seq, place // page], place % page
    # the cache holds k_out as it is, and V
    check_held(cache, before[0], [p.logical() for p in cache.k], where, got["k"], group, dtype, "K")
    check_held(cache, before[1], [p.logical() for p in cache.v], where, x["v"], group, dtype, "V")


@pytest.mark.parametrize("d,group", [(128, 0), (128, 64), (40, 20)])
@pytest.mark.parametrize("in_place", [True, False])
def test_append_positions_in_place_and_rows_without_a_place(ctx, d, group, in_place):
    rng = np.random.default_rng([8, d, group])
    # rows 0 and 9 belong to no sequence; sequence 0's first two rows lie in front of its cache; sequence 1
    # ends behind the page table; sequence 2's second page does not exist
    offsets, lengths, page = [1, 4, 6, 9], [1, 0, 18], 16
    cache = Cache(rng, [1, 1, 18], 2, d, page, capi.BFLOAT16, group)
    lengths[1] = cache.table.shape[1] * page + 1
    cache.table[1, -1] = cache.pool - 1  # (a spare page)
    assert cache.pool - 1 not in cache.table[[0, 2]]
    cache.table[2, 1] = cache.pool
    q, k, v = (rows_of(rng, [10, h, d], capi.BFLOAT16) for h in (4, 2, 2))
    x = {n: r.logical().astype(np.float64) for n, r in (("q", q), ("k", k), ("v", v))}
    before = [[p.logical() for p in c] for c in (cache.k, cache.v)]
    table = rotation_table(50, d // 4 * 2)
    positions = np.array([0, 3, 49, 7, 50, 11, 5, -1, 20, 0])
    got, _ = run_append(ctx, cache, lengths, offsets, k, v, q, table, positions, in_place=in_place)
    kept = np.array([1, 2, 3, 5, 6, 8])  # (rows 4 and 7 have positions that the table lacks)
    for n in ("q", "k"):
        check_turned(got[n][kept], x[n][kept], table, positions[kept], False, capi.BFLOAT16)
        assert np.isnan(got[n][[4, 7]]).all()
        assert (got[n][[0, 9]] == (x[n][[0, 9]] if in_place else SENTINEL)).all()
    # stored: row 3 of sequence 0 at place 0, row 5's place is behind the table, row 4 is the table's last but has no
    # position; sequence 2: row 6 at place 15, rows 7 and 8 in the page that is not there
    where = cache.table[[0, 2], [0, 0]], np.array([0, 15])
    check_held(cache, before[0], [p.logical() for p in cache.k], where, got["k"][[3, 6]], group, capi.BFLOAT16, "K")
    check_held(cache, before[1], [p.logical() for p in cache.v], where, x["v"][[3, 6]], group, capi.BFLOAT16, "V")


@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.HALF])
@pytest.mark.parametrize("d,group", [(128, 32), (64, 64), (60, 30)])
def test_append_groups_at_their_edges(ctx, dtype, d, group):
    # constant groups, zeros, one outlier, values that half rounds up, tiny and huge ones, infinities, NaN
    rng = np.random.default_rng([9, d])
    rows = np.stack([np.full(d, 0.3), np.zeros(d), np.where(np.arange(d) % group == 3, 1000.0, 0.001 * rng.standard_normal(d)),
                     100 + 0.01 * rng.standard_normal(d), 1e-6 * rng.standard_normal(d), -1e-8 * np.ones(d), 6e4 * np.sign(rng.standard_normal(d)),
                     (1e5 if dtype == capi.BFLOAT16 else 6.5e4) * rng.standard_normal(d).clip(-1, 1),
                     np.where(np.arange(d) == 5, np.inf, 1.0), np.where(np.arange(d) == 7, -np.inf, rng.standard_normal(d)),
                     np.where(np.arange(d) == d - 1, np.nan, 2.0), np.arange(d) % 16 - 7.5])[:, None]
    n = len(rows)
    cache = Cache(rng, [n], 1, d, 16, dtype, group)
    k, v = HT.from_logical(rows, dtype), HT.from_logical(-rows, dtype)
    before = [[p.logical() for p in c] for c in (cache.k, cache.v)]
    xk, xv = k.logical(), v.logical()
    run_append(ctx, cache, [n], [0, n], k, v, k_out=False)
    where = np.full(n, cache.table[0, 0]), np.arange(n)
    check_held(cache, before[0], [p.logical() for p in cache.k], where, xk, group, dtype, "K")
    check_held(cache, before[1], [p.logical() for p in cache.v], where, xv, group, dtype, "V")


def run_read(ctx, cache, lengths, offsets, dtype, t, how="dense"):
    outs = []
    d = capi.CacheReadDesc()
    for dim in (cache.d, cache.dv):
        dims = [t, cache.heads, dim]
        outs.append(HT.from_logical(np.full(dims, SENTINEL), dtype, rows_strides(dims, how)))
    d.k, d.v, d.cache = outs[0].desc(), outs[1].desc(), cache.desc()
    bufs = [o.upload(ctx) for o in outs]
    ctx.cache_read(d, cache.upload(ctx, lengths), ints(ctx, offsets), *bufs)
    return [o.fetch(ctx, b).logical() for o, b in zip(outs, bufs)]


@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.HALF, capi.FLOAT])
@pytest.mark.parametrize("d,page,group,order", [
    (128, 16, 0, (0, 1, 2, 3)), (128, 64, 64, (0, 2, 1, 3)), (64, 32, 32, (0, 1, 2, 3)), (64, 16, 0, (1, 0, 2, 3)),
    (128, 16, 128, (0, 1, 2, 3)), (80, 5, 20, (0, 1, 2, 3)), (72, 7, 0, (0, 2, 1, 3)), (128, 48, 32, (2, 0, 1, 3))])
def test_read(ctx, dtype, d, page, group, order):
    rng = np.random.default_rng([10, d, page])
    keys = [1, 0, 70, 16, 33]
    cache = Cache(rng, keys, 3, d, page, dtype, group, order=order)
    for rows, first in (([1, 0, 70, 16, 33], 0), ([1, 0, 5, 0, 20], 2)):  # all of them; the last ones, behind two rows of none
        offsets = starts(rows) + first
        got = run_read(ctx, cache, keys, offsets, dtype, offsets[-1] + 1, "wide" if d % 8 else "heads")
        for x, out in zip("kv", got):
            for b, n in enumerate(rows):
                ref = cache.rows(x, b)[keys[b] - n:]
                if group:  # low + scale code is exact in 64 bits: rounded in f32, then to the type
                    far = 2.0 ** -24 * np.abs(ref) + 0.5 * one_step(np.abs(ref) * (1 + 2.0 ** -24), dtype)
                    check(out[offsets[b]:offsets[b + 1]], ref, far)
                else:
                    assert np.array_equal(out[offsets[b]:offsets[b + 1]], ref)
            assert (out[:first] == SENTINEL).all() and (out[offsets[-1]:] == SENTINEL).all()


@pytest.mark.parametrize("group", [0, 64])
def test_read_rows_without_a_place(ctx, group):
    rng = np.random.default_rng([11, group])
    cache = Cache(rng, [3, 20, 2], 2, 128, 16, capi.BFLOAT16, group)
    lengths = [3, 20, cache.table.shape[1] * 16 + 2]
    cache.table[1, 0] = -1
    cache.table[2, -1] = 0
    k, v = run_read(ctx, cache, lengths, [0, 5, 9, 13], capi.BFLOAT16, 13)
    for out in (k, v):
        nan = np.isnan(out).all((1, 2))
        assert np.array_equal(nan, [True] * 2 + [False] * 7 + [False] * 2 + [True] * 2), nan
        assert np.isfinite(out[~nan]).all()


# ---- attention over pages --------------------------------------------------------
def run_paged(ctx, cache, lengths, q, offsets, causal=True, scale=None, o_how="dense", workspace=None):
    dims = [q.dims[0], q.dims[1], cache.dv]
    o = HT.from_logical(np.full(dims, SENTINEL), q.dtype, rows_strides(dims, o_how))
    d = capi.SdpaPagedDesc()
    d.q, d.o, d.cache, d.is_causal = q.desc(), o.desc(), cache.desc(), int(causal)
    if scale is not None:
        d.has_scale, d.scale = 1, scale
    bq, bo = q.upload(ctx), o.upload(ctx)
    ctx.sdpa_paged_fwd(d, cache.upload(ctx, lengths), bq, ints(ctx, offsets), bo)
    return o.fetch(ctx, bo).logical(), ctx.lib.fhip_sdpa_paged_fwd_supported(d)


def steps_of(cache, b, n):
    """attend()'s k_step and v_step of a cache in 4 bits."""
    if not cache.group:
        return {}
    j = np.arange(n)
    out = {}
    for x, pool in (("k_step", cache.k), ("v_step", cache.v)):
        pair = np.abs(pool[1].logical().astype(np.float64))[cache.table[b, j // cache.page], :, j % cache.page]
        scale, low = (np.repeat(pair[..., i::2], cache.group, -1) for i in (0, 1))
        out[x] = 143 * scale + low if x == "k_step" else 15 * scale
    return out


def check_paged(cache, lengths, q, offsets, got, causal=True, scale=None):
    ql = q.logical().astype(np.float64)
    for b, m in enumerate(lengths):
        r = slice(offsets[b], offsets[b + 1])
        n = offsets[b + 1] - offsets[b]
        seen = np.clip(m - n + 1 + np.arange(n), 0, m) if causal else np.full(n, m)
        ref, far = attend(ql[r], cache.rows("k", b, m), cache.rows("v", b, m), seen, q.dtype, scale, **steps_of(cache, b, m))
        check(got[r], ref, far, f"sequence {b}")
    assert (got[:offsets[0]] == SENTINEL).all() and (got[offsets[-1]:] == SENTINEL).all()


PAGED = [
    # keys, rows, query heads, key heads, page size
    ([1], [1], 1, 1, 16),
    ([5, 0, 33], [1, 1, 1], 4, 1, 16),         # a row that sees nothing
    ([16, 17, 31, 32], [1, 1, 1, 1], 8, 2, 16),
    ([300, 3, 64], [1, 0, 4], 8, 8, 32),
    ([1000, 40], [3, 5], 6, 2, 64),
    ([2, 129], [5, 17], 4, 2, 16),             # more rows than keys; a second tile of rows
    ([3000], [1], 7, 1, 48),
    ([700, 1, 90] * 9, [1, 1, 2] * 9, 4, 2, 128),
]


@pytest.mark.parametrize("keys,rows,hq,hkv,page", PAGED)
@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.HALF])
@pytest.mark.parametrize("d,group", [(64, 0), (128, 0), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_paged(ctx, keys, rows, hq, hkv, page, dtype, d, group):
    rng = np.random.default_rng([12, sum(keys), hq, d, group])
    cache = Cache(rng, keys, hkv, d, page, dtype, group)
    q = rows_of(rng, [sum(rows), hq, d], dtype, std=1.5)
    got, _ = run_paged(ctx, cache, keys, q, starts(rows))
    check_paged(cache, keys, q, starts(rows), got)


@pytest.mark.parametrize("dtype,d,dv,page,group", [
    (capi.FLOAT, 64, 64, 16, 0), (capi.FLOAT, 32, 48, 3, 16), (capi.BFLOAT16, 80, 80, 16, 0), (capi.HALF, 96, 96, 16, 96),
    (capi.BFLOAT16, 128, 128, 1, 0), (capi.HALF, 64, 64, 10, 64), (capi.BFLOAT16, 256, 256, 8, 128), (capi.BFLOAT16, 128, 128, 16, 16)])
def test_paged_other_sizes_types_and_pages(ctx, dtype, d, dv, page, group):
    rng = np.random.default_rng([13, d, page])
    keys, rows = [21, 0, 150], [2, 1, 3]
    cache = Cache(rng, keys, 2, d, page, dtype, group, dv)
    q = rows_of(rng, [6, 4, d], dtype)
    got, level = run_paged(ctx, cache, keys, q, starts(rows))
    assert level == 1
    check_paged(cache, keys, q, starts(rows), got)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("order", [(0, 2, 1, 3), (1, 0, 2, 3), (2, 1, 0, 3)])
def test_paged_layouts_scale_and_rows_of_no_sequence(ctx, d, group, causal, order):
    rng = np.random.default_rng([14, d, group])
    keys, offsets = [90, 1, 400], [2, 5, 6, 8]
    cache = Cache(rng, keys, 2, d, 16, capi.BFLOAT16, group, order=order)
    q = rows_of(rng, [11, 6, d], capi.BFLOAT16, "heads")
    got, _ = run_paged(ctx, cache, keys, q, offsets, causal, scale=-0.11, o_how="wide")
    check_paged(cache, keys, q, offsets, got, causal, scale=-0.11)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("page", [16, 32, 10])
def test_paged_what_no_row_sees_does_not_matter(ctx, d, group, page):
    # every place of the pool that holds no key is NaN, rows see only keys up to their own place
    rng = np.random.default_rng([15, d, page])
    keys, rows = [50, 7, 200], [3, 1, 20]
    cache = Cache(rng, keys, 2, d, page, capi.BFLOAT16, group)
    keep = np.zeros([cache.pool, cache.page], bool)
    for b, n in enumerate(keys):
        j = np.arange(n)
        keep[cache.table[b, j // page], j % page] = True
    for pool in (cache.k, cache.v):
        x = pool[-1].logical()
        x[~keep.repeat(1, 0)[:, None].repeat(2, 1)] = np.nan
        pool[-1] = HT(pool[-1].dims, pool[-1].strides, pool[-1].dtype, HT.from_logical(x, pool[-1].dtype).storage)
    q = rows_of(rng, [24, 4, d], capi.BFLOAT16)
    got, _ = run_paged(ctx, cache, keys, q, starts(rows))
    for b in range(3):
        keep_nan = cache.rows("k", b)
        assert np.isfinite(keep_nan).all()
    check_paged(cache, keys, q, starts(rows), got)


@pytest.mark.parametrize("group", [0, 64])
def test_paged_missing_pages_make_their_rows_nan(ctx, group):
    rng = np.random.default_rng([16, group])
    keys, rows = [40, 600, 20], [1, 2, 1]
    cache = Cache(rng, keys, 2, 128, 16, capi.BFLOAT16, group)
    q = rows_of(rng, [4, 8, 128], capi.BFLOAT16)
    cache.table[1, 20] = cache.pool + 5
    lengths = [40, 600, cache.table.shape[1] * 16 + 1]
    cache.table[2, :] = cache.table[0, 0]
    got, _ = run_paged(ctx, cache, lengths, q, starts(rows))
    assert np.isnan(got[1:]).all()
    ref, far = attend(q.logical().astype(np.float64)[:1], cache.rows("k", 0), cache.rows("v", 0), [40], capi.BFLOAT16, **steps_of(cache, 0, 40))
    check(got[:1], ref, far)


def test_paged_shares_pages(ctx):
    # two sequences with the same prefix in the same pages
    rng = np.random.default_rng([17])
    cache = Cache(rng, [70, 90], 2, 128, 16, capi.HALF)
    cache.table[1, :3] = cache.table[0, :3]
    q = rows_of(rng, [2, 8, 128], capi.HALF)
    got, _ = run_paged(ctx, cache, [70, 90], q, [0, 1, 2])
    check_paged(cache, [70, 90], q, [0, 1, 2], got)


# ---- together ----------------------------------------------------------------------
@pytest.mark.parametrize("group,d,dtype", [(0, 128, capi.BFLOAT16), (64, 128, capi.BFLOAT16), (32, 64, capi.HALF)])
def test_a_conversation(ctx, group, d, dtype):
    """Prompts go in and attend on each other, then a chunk behind them through the rows read back, then single tokens;
    the keys that later steps see are those that the cache holds."""
    rng = np.random.default_rng([18, d, group])
    page, hq, hkv = 16, 4, 2
    final = [50, 9, 131]
    cache = Cache(rng, final, hkv, d, page, dtype, group, fill=0.0)
    table = rotation_table(200, d)
    have = [0, 0, 0]
    for new in ([30, 5, 100], [16, 0, 28], [1, 1, 1], [3, 3, 2]):
        have = [h + n for h, n in zip(have, new)]
        at, t = starts(new), sum(new)
        q, k, v = (rows_of(rng, [t, h, d], dtype) for h in (hq, hkv, hkv))
        out, _ = run_append(ctx, cache, have, at, k, v, q, table)
        qo, ko = (HT.from_logical(out[n], dtype) for n in "qk")
        if have == new:  # whole prompts see the rows as they are
            got, _ = run_packed(ctx, qo, ko, v, at, True)
            check_packed(qo, ko, v, at, True, got)
        elif t > 10:
            kr, vr = run_read(ctx, cache, have, starts(have), dtype, sum(have))
            kr, vr = HT.from_logical(kr, dtype), HT.from_logical(vr, dtype)
            got, _ = run_packed(ctx, qo, kr, vr, at, True, kv_offsets=starts(have))
            check_packed(qo, kr, vr, at, True, got, kv_offsets=starts(have))
        got, _ = run_paged(ctx, cache, have, qo, at)
        check_paged(cache, have, qo, at, got)
    assert have == final


def test_graph_api():
    """Graphs that append and attend: a prompt, a chunk behind it, single tokens."""
    cpp_binary("test_serving_api", 120)
