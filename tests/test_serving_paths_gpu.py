"""Packed sequences and paged caches: which kernel a call gets, its other ways of cutting the
work, recorded graphs whose lengths and pages change between replays, large pools, workspaces."""
import ctypes

import numpy as np
import pytest
import torch  # (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
from serving import Cache, attend, check, rotation_table, starts
from test_serving_gpu import (check_packed, check_paged, ints, one_step, rows_of, run_append, run_packed, run_paged, run_read)

pytestmark = pytest.mark.gpu
BF16 = capi.BFLOAT16


# ---- which kernel ------------------------------------------------------------
@pytest.mark.parametrize("lens,hq,hkv,d,name", [
    ([40, 9], 4, 2, 64, "sdpa_packed d=64 causal=1 half"),
    ([1100], 4, 4, 128, "sdpa_packed d=128 causal=1 split"),
    ([4100], 32, 8, 128, "sdpa_packed d=128 causal=1"),
    ([4100], 32, 8, 64, "sdpa_packed d=64 causal=1 half"),
    ([4090], 16, 8, 64, "sdpa_packed d=64 causal=1 split"),
    ([700, 700, 700], 16, 8, 128, "sdpa_packed d=128 causal=1 half"),
    ([40, 9], 4, 2, 80, "sdpa_rows packed"),
])
def test_packed_route(ctx, lens, hq, hkv, d, name):
    rng = np.random.default_rng([30, d])
    t = sum(lens)
    q, k, v = (rows_of(rng, [t, h, d], BF16) for h in (hq, hkv, hkv))
    run_packed(ctx, q, k, v, starts(lens), True)
    assert ctx.last_kernel() == name


@pytest.mark.parametrize("keys,page,group,name", [
    ([90, 7], 16, 0, "sdpa_paged d=128 bits=16 group=0 cut=0"),
    ([90, 7], 32, 64, "sdpa_paged d=128 bits=4 group=64 cut=0"),
    ([3000, 7], 16, 0, "sdpa_paged d=128 bits=16 group=0 cut=1"),
    ([3000, 7], 16, 32, "sdpa_paged d=128 bits=4 group=32 cut=1"),
    ([90, 7], 8, 0, "sdpa_rows paged"),
])
def test_paged_route(ctx, keys, page, group, name):
    rng = np.random.default_rng([31, page, group])
    cache = Cache(rng, keys, 2, 128, page, BF16, group)
    run_paged(ctx, cache, keys, rows_of(rng, [2, 8, 128], BF16), [0, 1, 2])
    assert ctx.last_kernel().startswith(name), ctx.last_kernel()


@pytest.mark.parametrize("d,group,fast", [(128, 0, True), (64, 32, True), (192, 64, True), (80, 0, True), (36, 0, False), (40, 20, False)])
def test_cache_route(ctx, d, group, fast):
    rng = np.random.default_rng([32, d, group])
    cache = Cache(rng, [40, 5], 2, d, 16, BF16, group)
    k, v = (rows_of(rng, [7, 2, d], BF16) for _ in "kv")
    run_append(ctx, cache, [40, 5], [0, 4, 7], k, v)
    assert ctx.last_kernel().startswith("cache_append " if fast else "cache_append_rows"), ctx.last_kernel()
    run_read(ctx, cache, [40, 5], [0, 40, 45], BF16, 45)
    assert ctx.last_kernel().startswith("cache_read " if fast else "cache_read_rows"), ctx.last_kernel()


# ---- every way of cutting packed rows -------------------------------------------
@pytest.mark.parametrize("way", [0, 1, 2])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (capi.HALF, 128), (BF16, 64), (capi.HALF, 64)])
@pytest.mark.parametrize("lens,hq,hkv", [
    ([1], 3, 1), ([0, 5, 0, 0, 17, 1, 0], 4, 2), ([16] * 70, 2, 1), ([257, 2, 513, 31], 8, 2), ([700, 20], 5, 1), ([900], 1, 1)])
def test_packed_ways(ctx, knobs, way, causal, dtype, d, lens, hq, hkv):
    knobs(SDPA_PACKED=way)
    rng = np.random.default_rng([33, d, sum(lens), hq])
    t = sum(lens)
    q, k, v = rows_of(rng, [t, hq, d], dtype, std=2.0), rows_of(rng, [t, hkv, d], dtype), rows_of(rng, [t, hkv, d], dtype)
    got, _ = run_packed(ctx, q, k, v, starts(lens), causal)
    assert ctx.last_kernel() == f"sdpa_packed d={d} causal={int(causal)}" + ["", " split", " half"][way]
    check_packed(q, k, v, starts(lens), causal, got)


@pytest.mark.parametrize("way", [0, 1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_ways_behind_prefixes(ctx, knobs, way, d):
    knobs(SDPA_PACKED=way)
    rng = np.random.default_rng([34, d])
    lens, past = [3, 200, 0, 1, 64], [500, 0, 9, 129, 63]
    both = [a + b for a, b in zip(lens, past)]
    q, k, v = rows_of(rng, [sum(lens), 6, d], BF16, "fused"), rows_of(rng, [sum(both), 2, d], BF16), rows_of(rng, [sum(both), 2, d], BF16)
    got, _ = run_packed(ctx, q, k, v, starts(lens), True, starts(both))
    check_packed(q, k, v, starts(lens), True, got, starts(both))


# ---- more sequences than a wavefront or a workgroup has lanes ----------------------
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("batch", [65, 300])
def test_many_sequences(ctx, group, batch):
    rng = np.random.default_rng([35, batch, group])
    final = [int(x) for x in rng.integers(0, 40, batch)]
    new = [min(n, int(x)) for n, x in zip(final, rng.integers(0, 4, batch))]
    at, t, d = starts(new), sum(new), 64
    cache = Cache(rng, final, 2, d, 16, BF16, group)
    before = [cache.values(x).copy() for x in "kv"]
    q, k, v = (rows_of(rng, [t, h, d], BF16) for h in (4, 2, 2))
    run_append(ctx, cache, final, at, k, v, k_out=False)
    place = [(b, final[b] - new[b] + i) for b in range(batch) for i in range(new[b])]
    page = [cache.table[b, j // 16] for b, j in place], [j % 16 for _, j in place]
    for x, was, rows in zip("kv", before, (k, v)):
        now = cache.values(x)
        put = now[page[0], :, page[1]]
        ref = rows.logical().astype(np.float64)
        if group:  # half a scale, and a code of 15's part of the scale's and low's own roundings
            spread = ref.reshape(t, 2, -1, group)
            wide = np.repeat(spread.max(-1) - spread.min(-1), group, -1)
            low = np.repeat(np.abs(spread.min(-1)), group, -1)
            assert (np.abs(put - ref) <= wide / 15 * (0.5 + 2e-2) + (wide + low) * 2.0 ** -10).all()
        else:
            assert np.array_equal(put, ref)
        now[page[0], :, page[1]] = was[page[0], :, page[1]]
        assert np.array_equal(now, was), "other rows changed"
    got, _ = run_paged(ctx, cache, final, q, at)
    check_paged(cache, final, q, at, got)
    back = run_read(ctx, cache, final, starts(final), BF16, sum(final) + 1)
    for x, out in zip("kv", back):
        ref = np.concatenate([cache.rows(x, b) for b in range(batch)])
        far = 2.0 ** -24 * np.abs(ref) + 0.5 * one_step(np.abs(ref) * (1 + 2.0 ** -24), BF16) if group else 0 * ref
        check(out[:-1], ref, far)


@pytest.mark.parametrize("batch,most,past", [(65, 200, 0), (300, 90, 400), (1025, 9, 0), (5000, 3, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_packed_sequences(ctx, batch, most, past, causal):
    rng = np.random.default_rng([43, batch])
    new = [int(x) for x in rng.integers(0, most, batch)]
    keys = [n + int(x) for n, x in zip(new, rng.integers(0, past + 1, batch))]
    q, k, v = rows_of(rng, [sum(new), 2, 64], BF16), rows_of(rng, [sum(keys), 1, 64], BF16), rows_of(rng, [sum(keys), 1, 64], BF16)
    got, level = run_packed(ctx, q, k, v, starts(new), causal, starts(keys))
    assert level == 2
    check_packed(q, k, v, starts(new), causal, got, starts(keys))


def test_many_paged_sequences(ctx):
    rng = np.random.default_rng([44])
    keys, rows = [int(x) for x in rng.integers(0, 20, 5000)], [int(x) for x in rng.integers(0, 3, 5000)]
    cache = Cache(rng, keys, 1, 64, 16, BF16)
    q = rows_of(rng, [sum(rows), 2, 64], BF16)
    got, level = run_paged(ctx, cache, keys, q, starts(rows))
    assert level == 2
    for x in range(0, 5000, 61):  # (some of them: each takes the whole cache's values)
        a, b = starts(rows)[x], starts(rows)[x + 1]
        ref, far = attend(q.logical().astype(np.float64)[a:b], cache.rows("k", x), cache.rows("v", x),
                          np.clip(keys[x] - (b - a) + 1 + np.arange(b - a), 0, keys[x]), BF16)
        check(got[a:b], ref, far, f"sequence {x}")
    assert (got != 77).all()


def test_many_long_sequences(ctx):
    # more of them than pieces of the line, each worth several
    rng = np.random.default_rng([36])
    keys = [int(x) for x in rng.integers(1, 1400, 90)]
    cache = Cache(rng, keys, 1, 64, 32, capi.HALF)
    q = rows_of(rng, [90, 8, 64], capi.HALF)
    got, _ = run_paged(ctx, cache, keys, q, np.arange(91))
    check_paged(cache, keys, q, np.arange(91), got)


# ---- long ones ---------------------------------------------------------------------
@pytest.mark.parametrize("group", [0, 128])
def test_a_long_cache(ctx, group):
    rng = np.random.default_rng([37, group])
    keys = [150001, 3]
    cache = Cache(rng, keys, 1, 64 if not group else 128, 64, BF16, group)
    q = rows_of(rng, [3, 4, cache.d], BF16, std=2.0)
    got, _ = run_paged(ctx, cache, keys, q, [0, 2, 3])
    check_paged(cache, keys, q, [0, 2, 3], got)
    again, _ = run_paged(ctx, cache, keys, q, [0, 2, 3])
    assert np.array_equal(got, again)


@pytest.mark.parametrize("d", [64, 128])
def test_long_packed_rows(ctx, d):
    # few rows behind many keys, and the other way round
    rng = np.random.default_rng([38, d])
    q, k, v = rows_of(rng, [70, 4, d], BF16), rows_of(rng, [20010, 1, d], BF16), rows_of(rng, [20010, 1, d], BF16)
    got, _ = run_packed(ctx, q, k, v, [0, 65, 70], True, [0, 20000, 20010])
    check_packed(q, k, v, [0, 65, 70], True, got, [0, 20000, 20010])
    q, k, v = rows_of(rng, [3000, 2, d], BF16), rows_of(rng, [40, 1, d], BF16), rows_of(rng, [40, 1, d], BF16)
    got, _ = run_packed(ctx, q, k, v, [0, 2990, 3000], True, [0, 33, 40])
    check_packed(q, k, v, [0, 2990, 3000], True, got, [0, 33, 40])
    assert not got[:2957].any()


@pytest.mark.parametrize("group", [0, 64])
def test_a_pool_beyond_32_bits(group):
    """The same rows in a small pool and at the end of one of more than 2^32 bytes and 2^31 elements."""
    torch.manual_seed(3)
    c = capi.Context(0, torch.cuda.current_stream().cuda_stream)
    hk, page, d = 8, 64, 128
    row = d // 2 if group else d
    kind = torch.uint8 if group else torch.bfloat16
    small, large = 12, (1 << 32) // (hk * page * row) + 40
    keys = [600, 1]
    table = torch.zeros(2, 11, dtype=torch.int32, device="cuda")
    table[0, :10] = torch.arange(10, device="cuda") + 1
    lengths = torch.tensor(keys, dtype=torch.int32, device="cuda")
    news = torch.tensor([0, 5, 6], dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, 600, 601], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(6, hk, d, device="cuda", dtype=torch.bfloat16) for _ in "kv")
    q = torch.randn(6, 16, d, device="cuda", dtype=torch.bfloat16)
    codes = [torch.randint(0, 256, (small, hk, page, row), device="cuda", dtype=torch.uint8) if group else
             torch.randn(small, hk, page, row, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    params = [torch.rand(small, hk, page, 2 * d // group, device="cuda").half() for _ in "kv"] if group else []
    desc = lambda t: capi.TensorDesc.make(list(t.shape), list(t.stride()),  # noqa: E731
                                          {torch.uint8: capi.UINT8, torch.float16: capi.HALF, torch.bfloat16: BF16}[t.dtype])

    def run(pools, pairs, pages):
        cd = capi.CacheDesc()
        cd.k, cd.v = map(desc, pools)
        if group:
            cd.k_params, cd.v_params = map(desc, pairs)
        cd.batch, cd.pages_per_sequence, cd.page_stride = 2, 11, 11
        at = capi.CachePointers.make(*(t.data_ptr() for t in (*pools, pages, lengths, *pairs)))
        a, p, r = capi.CacheAppendDesc(), capi.SdpaPagedDesc(), capi.CacheReadDesc()
        a.k, a.v, a.cache = desc(k), desc(v), cd
        c.cache_append(a, at, k.data_ptr(), v.data_ptr(), news.data_ptr())
        o, ko, vo = torch.empty_like(q), *(torch.empty(601, hk, d, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        p.q, p.o, p.cache, p.is_causal = desc(q), desc(o), cd, 1
        space = torch.empty(c.sdpa_paged_workspace(p) + 256, device="cuda", dtype=torch.uint8)
        c.sdpa_paged_fwd(p, at, q.data_ptr(), news.data_ptr(), o.data_ptr(), (space.data_ptr() + 255) // 256 * 256)
        assert "sdpa_paged" in c.last_kernel()
        r.k, r.v, r.cache = desc(ko), desc(vo), cd
        c.cache_read(r, at, rows.data_ptr(), ko.data_ptr(), vo.data_ptr())
        torch.cuda.synchronize()
        return o, ko, vo

    shift = large - small
    far, far_pairs = [], []
    for x in codes:
        far.append(torch.empty(large, *x.shape[1:], device="cuda", dtype=kind))
        far[-1][shift:] = x
        if not group:
            assert far[-1].numel() > 1 << 31
        assert far[-1].numel() * far[-1].element_size() > 1 << 32
    for x in params:
        far_pairs.append(torch.empty(large, *x.shape[1:], device="cuda", dtype=torch.float16))
        far_pairs[-1][shift:] = x
    want = run(codes, params, table)
    got = run(far, far_pairs, table + shift)
    assert want[0].float().abs().max() > 0.01
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(codes + params, far + far_pairs):
        assert torch.equal(a, b[shift:])
    c.close()


@pytest.mark.parametrize("dtype", [BF16, capi.HALF])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_one_key_in_4_bits_is_its_value(ctx, dtype, d, group):
    """No probability is rounded where there is one key; of what acts on the codes, some eight roundings in f32 of at most
    143 scale + |low| are left, and the result's own."""
    rng = np.random.default_rng([46, d, group])
    cache = Cache(rng, [1] * 20, 2, d, 16, dtype, group)
    q = rows_of(rng, [20, 6, d], dtype)
    got, level = run_paged(ctx, cache, [1] * 20, q, np.arange(21))
    assert level == 2
    pair = np.abs(cache.v[1].logical().astype(np.float64))[cache.table[:, 0], :, 0]
    size = np.repeat(np.repeat(143 * pair[..., ::2] + pair[..., 1::2], group, -1), 3, 1)
    ref = np.repeat(np.stack([cache.rows("v", b)[0] for b in range(20)]), 3, 1)
    f32 = 8 * 2.0 ** -24 * size
    check(got, ref, f32 + 0.5 * one_step(np.abs(ref) + f32, dtype))


# ---- workspaces ------------------------------------------------------------------
def test_workspaces(ctx):
    rng = np.random.default_rng([39])
    keys = [3000, 7]
    cache = Cache(rng, keys, 2, 64, 16, BF16)
    q = rows_of(rng, [2, 4, 64], BF16)
    d = capi.SdpaPagedDesc()
    d.q = d.o = q.desc()
    d.cache, d.is_causal = cache.desc(), 1
    need = ctx.sdpa_paged_workspace(d)
    assert need > 0
    bq, bo, at, offsets, space = q.upload(ctx), q.upload(ctx), cache.upload(ctx), ints(ctx, [0, 1, 2]), ctx.alloc(need + 256)
    first = ctypes.cast(space.ptr, ctypes.c_void_p).value
    for where, size in ((first, need - 1), (first + 64, need), (None, need), (first, 0)):
        assert ctx.lib.fhip_sdpa_paged_fwd(ctx.handle, ctypes.byref(d), ctypes.byref(at), bq.ptr, offsets.ptr, bo.ptr, where, size) != 0
        assert f"needs {need} bytes of 256-byte aligned workspace" in ctx.lib.fhip_last_error(ctx.handle).decode()
    got = {}
    for fill in (0x00, 0xff):  # it holds nothing between calls, and nothing behind its end is touched
        space.upload(np.full(need + 256, fill, np.uint8))
        ctx.sdpa_paged_fwd(d, at, bq, offsets, bo, space)
        out = HT.from_logical(np.zeros(q.dims), BF16)
        got[fill] = out.fetch(ctx, bo).logical()
        assert (space.download(np.uint8, need + 256)[need:] == fill).all()
    assert np.array_equal(got[0], got[0xff])
    check_paged(cache, keys, q, [0, 1, 2], got[0])


def test_workspace_of_many_packed_sequences(ctx):
    rng = np.random.default_rng([45])
    lens = [int(x) for x in rng.integers(0, 30, 100)]
    q, k, v = (rows_of(rng, [sum(lens), h, 64], BF16) for h in (4, 2, 2))
    d = capi.SdpaPackedDesc()
    d.q = d.o = q.desc()
    d.k, d.v, d.batch, d.is_causal = k.desc(), v.desc(), 64, 1
    assert ctx.sdpa_packed_workspace(d) == 0
    d.batch = 100
    need = ctx.sdpa_packed_workspace(d)
    assert need > 0
    bufs, bo, offsets, space = [t.upload(ctx) for t in (q, k, v)], q.upload(ctx), ints(ctx, starts(lens)), ctx.alloc(need + 256)
    for where, size in ((space.ptr, need - 1), (space.ptr + 64, need), (None, need)):
        assert ctx.lib.fhip_sdpa_packed_fwd(ctx.handle, ctypes.byref(d), *(b.ptr for b in bufs), offsets.ptr, None, bo.ptr, where, size) != 0
        assert f"needs {need} bytes of 256-byte aligned workspace" in ctx.lib.fhip_last_error(ctx.handle).decode()
    for fill in (0x00, 0xff):
        space.upload(np.full(need + 256, fill, np.uint8))
        ctx.sdpa_packed_fwd(d, *bufs, offsets, bo, workspace=space)
        assert (space.download(np.uint8, need + 256)[need:] == fill).all()
        check_packed(q, k, v, starts(lens), True, HT.from_logical(np.zeros(q.dims), BF16).fetch(ctx, bo).logical())


# ---- recorded ----------------------------------------------------------------------
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("places", [256, 4096])
def test_steps_of_decoding_from_one_graph(group, places):
    """One graph of an append and the attention behind it, recorded on a context that has run nothing; lengths, rows,
    pages and who has a token change between the replays.  A second cache gets the same steps one by one."""
    torch.manual_seed(4)
    hq, hk, d, page, batch = 8, 2, 128, 16, 5
    table_len = places // page
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        gen = np.random.default_rng(40)
        pool = batch * table_len
        pages = torch.from_numpy(gen.permutation(pool).reshape(batch, table_len).astype(np.int32)).cuda()
        kind, row = (torch.uint8, d // 2) if group else (torch.bfloat16, d)
        first = [torch.zeros(pool, hk, page, row, device="cuda", dtype=kind) for _ in "kv"]
        pairs = [torch.zeros(pool, hk, page, 2 * d // group, device="cuda", dtype=torch.float16) for _ in "kv"] if group else []
        rotation = torch.from_numpy(rotation_table(places, d)).cuda()
        lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        offsets = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        q, k, v = (torch.zeros(8, h, d, device="cuda", dtype=torch.bfloat16) for h in (hq, hk, hk))
        types = {torch.uint8: capi.UINT8, torch.float16: capi.HALF, torch.bfloat16: BF16, torch.float32: capi.FLOAT}
        desc = lambda t: capi.TensorDesc.make(list(t.shape), list(t.stride()), types[t.dtype])  # noqa: E731

        def make():
            pools, pp = [t.clone() for t in first], [t.clone() for t in pairs]
            cd = capi.CacheDesc()
            cd.k, cd.v = map(desc, pools)
            if group:
                cd.k_params, cd.v_params = map(desc, pp)
            cd.batch, cd.pages_per_sequence, cd.page_stride = batch, table_len, table_len
            at = capi.CachePointers.make(*(t.data_ptr() for t in (*pools, pages, lengths, *pp)))
            qo, o = torch.zeros_like(q), torch.zeros_like(q)
            a, p = capi.CacheAppendDesc(), capi.SdpaPagedDesc()
            a.k, a.v, a.q, a.q_out, a.rotation, a.cache = desc(k), desc(v), desc(q), desc(qo), desc(rotation), cd
            p.q, p.o, p.cache, p.is_causal = desc(qo), desc(o), cd, 1
            c = capi.Context(0, stream.cuda_stream)
            space = torch.empty(c.sdpa_paged_workspace(p), device="cuda", dtype=torch.uint8)

            def call():
                c.cache_append(a, at, k.data_ptr(), v.data_ptr(), offsets.data_ptr(), q=q.data_ptr(),
                               rotation=rotation.data_ptr(), q_out=qo.data_ptr())
                c.sdpa_paged_fwd(p, at, qo.data_ptr(), offsets.data_ptr(), o.data_ptr(), space.data_ptr())
            return c, call, o, pools + pp, space

        one, call_one, o_one, pools_one, keep_one = make()
        two, call_two, o_two, pools_two, keep_two = make()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call_one()
        have = np.zeros(batch, np.int64)
        for step in range(12):
            new = gen.integers(0, 3, batch)
            new[step % batch] = 0
            while new.sum() > 8:
                new[new.argmax()] -= 1
            if step == 5:  # sequences that have grown by many tokens meanwhile
                have = have + gen.integers(0, places - 60, batch)
            have = np.minimum(have + new, places)
            lengths.copy_(torch.from_numpy(have.astype(np.int32)))
            offsets.copy_(torch.from_numpy(starts(new).astype(np.int32)))
            if step == 8:  # a page moves
                spare = pages[0, 0].clone()
                pages[0, 0] = pages[1, table_len - 1]
                pages[1, table_len - 1] = spare
            for t in (q, k, v):
                t.copy_(torch.randn_like(t))
            o_one.fill_(5), o_two.fill_(5)
            graph.replay()
            call_two()
            stream.synchronize()
            assert torch.equal(o_one, o_two), step
            assert all(torch.equal(a, b) for a, b in zip(pools_one, pools_two)), step
            assert bool((o_one[int(new.sum()):] == 5).all())
            assert bool(torch.isfinite(o_one.float()).all())
        del graph
        one.close(), two.close()


def test_two_graphs_that_share_a_workspace():
    """Recorded one after the other, replayed in turn on one stream: each finds the workspace as the other left it."""
    torch.manual_seed(5)
    hq, hk, d, page, places = 8, 2, 64, 16, 4096
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = capi.Context(0, stream.cuda_stream)
        desc = lambda t: capi.TensorDesc.make(list(t.shape), list(t.stride()), BF16)  # noqa: E731
        calls, space = [], None
        for batch, seed in ((3, 1), (1, 2)):
            pages = torch.randperm(batch * places // page, device="cuda").to(torch.int32).reshape(batch, -1)
            pools = [torch.randn(batch * places // page, hk, page, d, device="cuda").bfloat16() for _ in "kv"]
            lengths = torch.randint(1, places, (batch,), device="cuda", dtype=torch.int32)
            offsets = torch.arange(batch + 1, device="cuda", dtype=torch.int32)
            q, o = torch.randn(batch, hq, d, device="cuda").bfloat16(), torch.zeros(batch, hq, d, device="cuda").bfloat16()
            p = capi.SdpaPagedDesc()
            p.q, p.o, p.is_causal = desc(q), desc(o), 1
            p.cache.k, p.cache.v = map(desc, pools)
            p.cache.batch, p.cache.pages_per_sequence, p.cache.page_stride = batch, places // page, places // page
            if space is None:
                space = torch.empty(c.sdpa_paged_workspace(p), device="cuda", dtype=torch.uint8)
            assert c.sdpa_paged_workspace(p) <= space.numel()
            at = capi.CachePointers.make(pools[0].data_ptr(), pools[1].data_ptr(), pages.data_ptr(), lengths.data_ptr())
            call = lambda p=p, at=at, q=q, offsets=offsets, o=o, hold=pools + [pages]: c.sdpa_paged_fwd(  # noqa: E731
                p, at, q.data_ptr(), offsets.data_ptr(), o.data_ptr(), space.data_ptr())
            graph = torch.cuda.CUDAGraph()
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                call()
            calls.append((graph, call, q, o, lengths))
        for i in range(6):
            for graph, call, q, o, lengths in calls:
                q.copy_(torch.randn_like(q))
                lengths.copy_(torch.randint(1, places, lengths.shape, device="cuda", dtype=torch.int32))
                call()
                o_want = o.clone()
                o.zero_()
                graph.replay()
                assert torch.equal(o, o_want), i
            for graph, _, _, o, _ in calls:
                o.zero_()
                graph.replay()
            stream.synchronize()
            assert bool((calls[0][3] != 0).any()) and torch.equal(calls[1][3], o_want)
        del graph, calls
        c.close()


@pytest.mark.parametrize("d", [64, 128])
def test_packed_from_a_graph(d):
    torch.manual_seed(6)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        one, two = (capi.Context(0, stream.cuda_stream) for _ in "ab")
        q, k, v = (torch.randn(900, h, d, device="cuda").bfloat16() for h in (8, 2, 2))
        outs = [torch.zeros_like(q) for _ in "ab"]
        offsets = torch.zeros(7, device="cuda", dtype=torch.int32)
        p = capi.SdpaPackedDesc()
        p.q = p.o = capi.TensorDesc.make([900, 8, d], [8 * d, d, 1], BF16)
        p.k = p.v = capi.TensorDesc.make([900, 2, d], [2 * d, d, 1], BF16)
        p.batch, p.is_causal = 6, 1
        call = lambda c, o: c.sdpa_packed_fwd(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), offsets.data_ptr(), o.data_ptr())  # noqa: E731
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call(one, outs[0])
        for lens in ([900, 0, 0, 0, 0, 0], [1, 2, 3, 4, 5, 6], [0] * 6, [100, 300, 7, 0, 200, 293], [150] * 6):
            offsets.copy_(torch.from_numpy(starts(lens)))
            q.copy_(torch.randn_like(q))
            for o in outs:
                o.fill_(3)
            graph.replay()
            call(two, outs[1])
            stream.synchronize()
            assert torch.equal(*outs) and bool((outs[0][sum(lens):] == 3).all())
        del graph
        one.close(), two.close()


# ---- metadata that does not fit the tensors ------------------------------------------
@pytest.mark.parametrize("d", [64, 80])
def test_offsets_behind_the_rows(ctx, d):
    """The last sequence claims more rows than there are: the others, and memory behind the tensors, do not notice."""
    rng = np.random.default_rng([41, d])
    q, k, v = rows_of(rng, [90, 4, d], BF16), rows_of(rng, [90, 2, d], BF16), rows_of(rng, [90, 2, d], BF16)
    dims = [90 + 64, 4, d]
    o = HT.from_logical(np.full(dims, 3.0), BF16)
    desc = capi.SdpaPackedDesc()
    desc.q, desc.k, desc.v = q.desc(), k.desc(), v.desc()
    desc.o = capi.TensorDesc.make([90, 4, d], [4 * d, d, 1], BF16)
    desc.batch, desc.is_causal = 3, 1
    buf = o.upload(ctx)
    ctx.sdpa_packed_fwd(desc, q.upload(ctx), k.upload(ctx), v.upload(ctx), ints(ctx, [0, 40, 50, 5000]), buf)
    got = o.fetch(ctx, buf).logical()
    assert (got[90:] == 3).all()
    got[50:] = 77.0  # (rows of the third sequence, which the checks take for rows of none)
    check_packed(q, k, v, [0, 40, 50], True, got[:90])

    cache = Cache(rng, [40, 30, 20], 2, d, 16, BF16)
    desc = capi.SdpaPagedDesc()
    desc.q, desc.cache, desc.is_causal = q.desc(), cache.desc(), 1
    desc.o = capi.TensorDesc.make([90, 4, d], [4 * d, d, 1], BF16)
    buf = HT.from_logical(np.full(dims, 3.0), BF16).upload(ctx)
    ctx.sdpa_paged_fwd(desc, cache.upload(ctx), q.upload(ctx), ints(ctx, [0, 1, 3, 5000]), buf)
    got = o.fetch(ctx, buf).logical()
    assert (got[90:] == 3).all()
    got[3:] = 77.0
    check_paged(cache, [40, 30], q, [0, 1, 3], got[:90])

    read = capi.CacheReadDesc()
    read.k = read.v = capi.TensorDesc.make([60, 2, d], [2 * d, d, 1], BF16)
    read.cache = cache.desc()
    bufs = [HT.from_logical(np.full([100, 2, d], 3.0), BF16) for _ in "kv"]
    at = [b.upload(ctx) for b in bufs]
    ctx.cache_read(read, cache.upload(ctx), ints(ctx, [0, 40, 50, 5000]), *at)
    for x, host, b in zip("kv", bufs, at):
        out = host.fetch(ctx, b).logical()
        assert np.array_equal(out[:40], cache.rows(x, 0)) and np.array_equal(out[40:50], cache.rows(x, 1)[20:])
        assert np.isnan(out[50:60]).all() and (out[60:] == 3).all()  # (places in front of the first)


@pytest.mark.parametrize("lengths", [[-5, 20, 30], [40, 20, 2 ** 30]])
def test_lengths_that_no_cache_has(ctx, lengths):
    rng = np.random.default_rng([42])
    cache = Cache(rng, [40, 20, 30], 2, 128, 16, BF16)
    q = rows_of(rng, [3, 8, 128], BF16)
    got, _ = run_paged(ctx, cache, lengths, q, [0, 1, 2, 3])
    ok = [b for b in range(3) if 0 <= lengths[b] <= 40]
    for b in ok:
        one = np.full_like(got, 77.0)
        one[b] = got[b]
        check_paged(cache, [0] * b + [lengths[b]], q, [b] * (b + 1) + [b + 1], one)
    if lengths[0] < 0:
        assert not got[0].any()  # no key: 0
    else:
        assert np.isnan(got[2]).all()  # keys that the table has no places for


# ---- heads and pointers ------------------------------------------------------------
@pytest.mark.parametrize("hq,hk", [(40, 1), (66, 2), (17, 17)])
@pytest.mark.parametrize("group", [0, 64])
def test_many_heads(ctx, hq, hk, group):
    rng = np.random.default_rng([47, hq, group])
    lens, past = [9, 1, 0, 30], [70, 0, 5, 2]
    keys = [a + b for a, b in zip(lens, past)]
    cache = Cache(rng, keys, hk, 64, 16, BF16, group)
    q = rows_of(rng, [40, hq, 64], BF16)
    got, level = run_paged(ctx, cache, keys, q, starts(lens))
    assert level == 2
    check_paged(cache, keys, q, starts(lens), got)
    k, v = rows_of(rng, [sum(keys), hk, 64], BF16), rows_of(rng, [sum(keys), hk, 64], BF16)
    got, level = run_packed(ctx, q, k, v, starts(lens), True, starts(keys))
    assert level == 2
    check_packed(q, k, v, starts(lens), True, got, starts(keys))


@pytest.mark.parametrize("group", [0, 32])
def test_tensors_on_odd_addresses(ctx, group):
    """One element behind where the vector kernels can load: the general ones take the call."""
    rng = np.random.default_rng([48, group])
    keys, new, d = [30, 7], [3, 2], 64
    at = starts(new)
    cache = Cache(rng, keys, 2, d, 16, BF16, group)
    tensors = {n: rows_of(rng, [5, h, d], BF16) for n, h in (("q", 4), ("k", 2), ("v", 2))}

    def shifted(t):
        raw = np.concatenate([np.zeros(1, t.storage.dtype), t.storage.reshape(-1)])
        buf = ctx.to_device(raw)
        return buf, buf.ptr + raw.itemsize

    bufs = {n: shifted(t) for n, t in tensors.items()}
    offsets, pointers = ints(ctx, at), cache.upload(ctx)
    a = capi.CacheAppendDesc()
    a.k, a.v, a.cache = tensors["k"].desc(), tensors["v"].desc(), cache.desc()
    ctx.cache_append(a, pointers, bufs["k"][1], bufs["v"][1], offsets)
    assert ctx.last_kernel() == "cache_append_rows"
    cache.fetch(ctx)
    if not group:
        for b, n in enumerate(keys):
            assert np.array_equal(cache.rows("k", b)[n - new[b]:], tensors["k"].logical()[at[b]:at[b + 1]])
    out = HT.from_logical(np.full([5, 4, d], 77.0), BF16)
    p = capi.SdpaPagedDesc()
    p.q, p.o, p.cache, p.is_causal = tensors["q"].desc(), out.desc(), cache.desc(), 1
    bo = out.upload(ctx)
    ctx.sdpa_paged_fwd(p, pointers, bufs["q"][1], offsets, bo)
    assert ctx.last_kernel() == "sdpa_rows paged"
    check_paged(cache, keys, tensors["q"], at, out.fetch(ctx, bo).logical())
    s = capi.SdpaPackedDesc()
    s.q, s.k, s.v, s.o = (tensors[n].desc() for n in "qkvq")
    s.batch, s.is_causal = 2, 1
    bo = HT.from_logical(np.full([5, 4, d], 77.0), BF16).upload(ctx)
    ctx.sdpa_packed_fwd(s, *(bufs[n][1] for n in "qkv"), offsets, bo)
    assert ctx.last_kernel() == "sdpa_rows packed"
    check_packed(tensors["q"], tensors["k"], tensors["v"], at, True, out.fetch(ctx, bo).logical())
    r = capi.CacheReadDesc()
    r.k = r.v = capi.TensorDesc.make([37, 2, d], [2 * d, d, 1], BF16)
    r.cache = cache.desc()
    room = [ctx.alloc(2 * (37 * 2 * d + 1)) for _ in "kv"]
    ctx.cache_read(r, pointers, ints(ctx, starts(keys)), *(b.ptr + 2 for b in room))
    assert ctx.last_kernel() == "cache_read_rows"
    for x, b in zip("kv", room):
        back = HT([37, 2, d], [2 * d, d, 1], BF16, b.download(np.uint16)[1:].copy()).logical()
        ref = np.concatenate([cache.rows(x, i) for i in range(2)])
        far = 2.0 ** -24 * np.abs(ref) + 0.5 * one_step(np.abs(ref) * (1 + 2.0 ** -24), BF16) if group else 0 * ref
        check(back, ref, far)
