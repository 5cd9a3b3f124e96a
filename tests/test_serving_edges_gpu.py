"""Packed sequences and paged caches at their edges: metadata of any value, sizes at the limit of a launch, long
lines of pieces, small and infinite values."""
import numpy as np
import pytest
import torch  # (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
import test_serving_paths_gpu
from serving import Cache, attend, check
from test_serving_gpu import check_held, check_paged, ints, rows_of, run_packed, run_paged, steps_of

pytestmark = pytest.mark.gpu
BF16 = capi.BFLOAT16
INT_MIN = -2 ** 31


def widened(cache, room):
    """The cache's table with room for `room` keys, whose further entries are never read."""
    more = room // cache.page - cache.table.shape[1]
    if more > 0:
        cache.table = np.concatenate([cache.table, np.full([len(cache.keys), more], -7, np.int32)], 1)
    return cache


# ---- metadata of any value -------------------------------------------------------
class Guarded:
    """A packed tensor between 64 rows in front and behind that nobody may touch."""

    def __init__(self, ctx, t, heads, d):
        self.host = HT.from_logical(np.full([t + 128, heads, d], 3.0), BF16)
        self.buf, self.t = self.host.upload(ctx), t
        self.ptr = self.buf.ptr + 64 * heads * d * 2
        self.desc = capi.TensorDesc.make([t, heads, d], [heads * d, d, 1], BF16)

    def fetch(self, ctx):
        out = self.host.fetch(ctx, self.buf).logical()
        assert (out[:64] == 3).all() and (out[64 + self.t:] == 3).all(), "rows outside the tensor were written"
        return out[64:64 + self.t]


@pytest.mark.parametrize("d,more", [(64, 0), (128, 0), (80, 0), (64, 70)])  # (70: more sequences than lanes)
@pytest.mark.parametrize("room", [64, 2048])
@pytest.mark.parametrize("offsets,alone", [
    ([5, INT_MIN, 20, 30], (2, 20, 30)),               # (sequence, rows that no other one claims)
    ([0, 10, -7, 20, 15, 60], (4, 20, 60)),
    ([7, INT_MIN, INT_MIN + 3, -1, 0, 30], (4, 7, 30)),
    ([INT_MIN, INT_MIN, 2 ** 31 - 1, 2 ** 31 - 1], None),
])
def test_offsets_of_any_value(ctx, d, more, room, offsets, alone):
    """Rows that one sequence alone claims are right, memory outside the tensors and the workspace is not touched."""
    rng = np.random.default_rng([50, d, room])
    offsets = offsets + offsets[-1:] * more
    t, batch = 90, len(offsets) - 1
    keys = [int(x) for x in rng.integers(40, 60, batch)]
    cache = widened(Cache(rng, keys, 2, d, 16, BF16), room)
    q, k, v = (rows_of(rng, [t, h, d], BF16) for h in (4, 2, 2))
    bufs, at, cached = [x.upload(ctx) for x in (q, k, v)], ints(ctx, offsets), cache.upload(ctx)
    p = capi.SdpaPagedDesc()
    o = Guarded(ctx, t, 4, d)
    p.q, p.o, p.cache, p.is_causal = q.desc(), o.desc, cache.desc(), 1
    need = ctx.sdpa_paged_workspace(p)
    space = ctx.to_device(np.full(need + 4096, 0x5a, np.uint8))
    ctx.sdpa_paged_fwd(p, cached, bufs[0], at, o.ptr, space)
    assert (space.download(np.uint8)[need:] == 0x5a).all()
    got = o.fetch(ctx)
    ql, kl, vl = (x.logical().astype(np.float64) for x in (q, k, v))
    if alone:
        b, lo, hi = alone
        n = offsets[b + 1] - max(offsets[b], 0)
        seen = np.clip(keys[b] - n + 1 + np.arange(n), 0, keys[b])
        ref, far = attend(ql[hi - n:hi], cache.rows("k", b), cache.rows("v", b), seen, BF16)
        check(got[lo:hi], ref[lo - hi:], far[lo - hi:], "paged")
    o = Guarded(ctx, t, 4, d)
    s = capi.SdpaPackedDesc()
    s.q, s.k, s.v, s.o, s.batch, s.is_causal = q.desc(), k.desc(), v.desc(), o.desc, batch, 1
    ctx.sdpa_packed_fwd(s, *bufs, at, o.ptr)
    got = o.fetch(ctx)
    if alone:
        ref, far = attend(ql[hi - n:hi], kl[hi - n:hi], vl[hi - n:hi], np.arange(n) + 1, BF16)
        check(got[lo:hi], ref[lo - hi:], far[lo - hi:], "packed")
    r = capi.CacheReadDesc()
    outs = [Guarded(ctx, t, 2, d) for _ in "kv"]
    r.k, r.v, r.cache = outs[0].desc, outs[1].desc, cache.desc()
    ctx.cache_read(r, cached, at, *(x.ptr for x in outs))
    for x, out in zip("kv", outs):
        got = out.fetch(ctx)
        if alone:  # (row hi - 1 has the sequence's last place)
            assert np.array_equal(got[lo:hi], cache.rows(x, b)[keys[b] - (hi - lo):])
    a = capi.CacheAppendDesc()
    a.k, a.v, a.cache = k.desc(), v.desc(), cache.desc()
    ctx.cache_append(a, cached, bufs[1], bufs[2], at)
    cache.fetch(ctx)
    if alone:
        assert np.array_equal(cache.rows("v", b)[keys[b] - (hi - lo):], vl[lo:hi])


# ---- more workgroups than one dimension of a grid holds ---------------------------------
def desc_of(t, strides=None):
    types = {torch.bfloat16: BF16, torch.float32: capi.FLOAT, torch.float16: capi.HALF}
    return capi.TensorDesc.make(list(t.shape), list(t.stride() if strides is None else strides), types[t.dtype])


def pages_of(k, v, table, lengths):
    c = capi.CacheDesc()
    c.k, c.v = desc_of(k), desc_of(v)
    c.batch, c.pages_per_sequence = table.shape
    c.page_stride = table.shape[1]
    return c, capi.CachePointers.make(*(t.data_ptr() for t in (k, v, table, lengths)))


def cuda_ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


@pytest.fixture
def own_stream():
    """A context on the stream that torch's work of the test is on as well (of the null stream it would make its own)."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = capi.Context(0, stream.cuda_stream)
        yield c
        stream.synchronize()
        c.close()
    torch.cuda.empty_cache()


def test_append_and_read_of_2_to_the_26_rows_of_heads(own_stream):
    """The general kernels: one wavefront per row of a head, 2^32 threads and some more."""
    c, t, page = own_stream, (1 << 25) + 3, 1 << 16
    k, v = (torch.randn(t, 1, 2, device="cuda") for _ in "kv")
    pools = [torch.zeros(t // page + 1, 1, page, 2, device="cuda") for _ in "kv"]
    table = torch.arange(t // page + 1, device="cuda", dtype=torch.int32)[None]
    lengths, offsets = cuda_ints([t]), cuda_ints([0, t])
    cache, at = pages_of(*pools, table, lengths)
    a = capi.CacheAppendDesc()
    a.k, a.v, a.cache = desc_of(k), desc_of(v), cache
    c.cache_append(a, at, k.data_ptr(), v.data_ptr(), offsets.data_ptr())
    assert c.last_kernel() == "cache_append_rows"
    for x, pool in zip((k, v), pools):
        assert torch.equal(pool.view(-1, 1, 2)[:t], x) and not pool.view(-1, 2)[t:].any()
    back = [torch.zeros_like(x) for x in (k, v)]
    r = capi.CacheReadDesc()
    r.k, r.v, r.cache = desc_of(k), desc_of(v), cache
    c.cache_read(r, at, offsets.data_ptr(), *(x.data_ptr() for x in back))
    assert c.last_kernel() == "cache_read_rows"
    assert torch.equal(back[0], k) and torch.equal(back[1], v)


def test_append_of_many_wide_rows(own_stream):
    """The kernel of 16-bit rows, 64 lanes a row: every row is the same (a stride of 0) and goes to one page, but for the
    last, which alone lies in another one."""
    c, t, page, d = own_stream, (1 << 26) + 1, 1 << 14, 512
    k, v = (torch.randn(1, 1, d, device="cuda").bfloat16() for _ in "kv")
    pools = [torch.zeros(2, 1, page, d, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    table = torch.zeros(1, t // page + 1, device="cuda", dtype=torch.int32)
    table[0, -1] = 1
    lengths, offsets = cuda_ints([t]), cuda_ints([0, t])
    cache, at = pages_of(*pools, table, lengths)
    a = capi.CacheAppendDesc()
    a.k = a.v = capi.TensorDesc.make([t, 1, d], [0, d, 1], BF16)
    a.cache = cache
    c.cache_append(a, at, k.data_ptr(), v.data_ptr(), offsets.data_ptr())
    assert c.last_kernel().startswith("cache_append bits=16 lanes=64")
    for x, pool in zip((k, v), pools):
        assert torch.equal(pool[0, 0], x[0].expand(page, d))
        assert torch.equal(pool[1, 0, :1], x[0]) and not pool[1, 0, 1:].any()


def test_read_of_2_to_the_29_rows(own_stream):
    """The kernel of 16-bit rows, 8 lanes a row.  All pages but the last are one."""
    c, t, page, d = own_stream, (1 << 29) + 1, 1 << 16, 8
    pools = [torch.randn(2, 1, page, d, device="cuda").bfloat16() for _ in "kv"]
    table = torch.zeros(1, t // page + 1, device="cuda", dtype=torch.int32)
    table[0, -1] = 1
    lengths, offsets = cuda_ints([t]), cuda_ints([0, t])
    cache, at = pages_of(*pools, table, lengths)
    outs = [torch.zeros(t, 1, d, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    r = capi.CacheReadDesc()
    r.k, r.v, r.cache = desc_of(outs[0]), desc_of(outs[1]), cache
    c.cache_read(r, at, offsets.data_ptr(), *(x.data_ptr() for x in outs))
    assert c.last_kernel().startswith("cache_read bits=16 lanes=8")
    for pool, out in zip(pools, outs):
        assert bool((out[:-1].view(-1, page, d) == pool[0, 0]).all()) and torch.equal(out[-1], pool[1, :, 0])


@pytest.mark.parametrize("d,level", [(2, 1), (64, 2)])
def test_packed_rows_of_2_to_the_24_tiles(own_stream, d, level):
    """Sequences of one row each: what they see is their own V.  (K and V of all heads are one, by a stride of 0.)"""
    c, heads = own_stream, 64
    t = (1 << 20) + 1 if level == 1 else (1 << 18) + 1
    kind = torch.float32 if level == 1 else torch.bfloat16
    q, o = torch.randn(t, heads, d, device="cuda", dtype=kind), torch.zeros(t, heads, d, device="cuda", dtype=kind)
    k, v = (torch.randn(t, 1, d, device="cuda", dtype=kind) for _ in "kv")
    offsets = torch.arange(t + 1, device="cuda", dtype=torch.int32)
    p = capi.SdpaPackedDesc()
    p.q, p.o, p.batch, p.is_causal = desc_of(q), desc_of(o), t, 1
    p.k = p.v = capi.TensorDesc.make([t, heads, d], [d, 0, 1], p.q.dtype)
    assert c.lib.fhip_sdpa_packed_fwd_supported(p) == level
    space = torch.empty(c.sdpa_packed_workspace(p) + 256, device="cuda", dtype=torch.uint8)
    c.sdpa_packed_fwd(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), offsets.data_ptr(), o.data_ptr(), workspace=(space.data_ptr() + 255) // 256 * 256)
    assert c.last_kernel().startswith("sdpa_packed" if level == 2 else "sdpa_rows")
    assert bool((o == v).all())


def test_paged_rows_of_2_to_the_24_tiles(own_stream):
    """Sequences of one row and one key, all in the same page."""
    c, heads, t, d = own_stream, 64, (1 << 18) + 1, 64
    q, o = (torch.randn(t, heads, d, device="cuda", dtype=torch.bfloat16) for _ in "qo")
    pools = [torch.randn(1, heads, 16, d, device="cuda").bfloat16() for _ in "kv"]
    table, lengths = torch.zeros(t, 1, device="cuda", dtype=torch.int32), torch.ones(t, device="cuda", dtype=torch.int32)
    offsets = torch.arange(t + 1, device="cuda", dtype=torch.int32)
    p = capi.SdpaPagedDesc()
    p.q, p.o, p.is_causal = desc_of(q), desc_of(o), 1
    p.cache, at = pages_of(*pools, table, lengths)
    assert c.lib.fhip_sdpa_paged_fwd_supported(p) == 2
    space = torch.empty(c.sdpa_paged_workspace(p) + 256, device="cuda", dtype=torch.uint8)
    c.sdpa_paged_fwd(p, at, q.data_ptr(), offsets.data_ptr(), o.data_ptr(), (space.data_ptr() + 255) // 256 * 256)
    assert c.last_kernel().startswith("sdpa_paged d=64")
    assert bool((o == pools[1][0, :, 0]).all())


# ---- 4 bits of any size -----------------------------------------------------------
class Given:
    """The values that a pool is made of, in the place of a generator."""

    def __init__(self, values):
        self.values = values

    def standard_normal(self, dims):
        return np.broadcast_to(self.values, dims)


@pytest.mark.parametrize("dtype", [capi.HALF, BF16])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("keys,room", [([700, 3, 90], 0), ([3000, 40], 4096)])
@pytest.mark.parametrize("how", ["1e-3", "1e-4", "1e-5", "3e3", "rows", "groups", "rising", "falling", "constant"])
def test_values_in_4_bits_of_any_size(ctx, dtype, d, group, keys, room, how):
    """P times V's scale is rounded to the rows' type: it has to keep that type's bits for scales from half's smallest to
    its largest, also where they change along the keys while the maximum moves, or from group to group."""
    rng = np.random.default_rng([51, d, group, sum(keys)])
    cache = Cache(rng, keys, 2, d, 16, dtype, group)
    at = np.zeros([cache.pool, 1, 16, 1])  # each place's part of its sequence
    for b, n in enumerate(keys):
        j = np.arange(n)
        at[cache.table[b, j // 16], 0, j % 16, 0] = j / n
    size = {"rows": 10.0 ** rng.uniform(-5, 2, at.shape), "rising": 10.0 ** (-5 + 8 * at), "falling": 10.0 ** (3 - 8 * at),
            "groups": np.repeat(10.0 ** rng.uniform(-3, 1, [1, 2, 1, d // group]), group, -1), "constant": 0.0}.get(how)
    v = rng.standard_normal([cache.pool, 2, 16, d]) * (float(how) if size is None else size) + (0.3 if how == "constant" else 0)
    cache.v = cache._pool(Given(v), d, None)
    if how in ("rising", "falling"):  # scores that rise along the keys by e^40, so that the last ones count
        k = rng.standard_normal([cache.pool, 2, 16, d]) * 0.2 + 40 * at / np.sqrt(d)
        cache.k = cache._pool(Given(k), d, None)
    widened(cache, room)
    q = rows_of(rng, [2 * len(keys), 4, d], dtype, std=1.0)
    if how in ("rising", "falling"):
        q = HT.from_logical(1.0 + 0.01 * q.logical(), dtype)
    offsets = 2 * np.arange(len(keys) + 1)
    got, level = run_paged(ctx, cache, keys, q, offsets)
    assert level == 2
    check_paged(cache, keys, q, offsets, got)


# ---- scores of -inf ---------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("room", [64, 4096])
def test_keys_of_minus_infinity(ctx, d, room):
    """A key with a score of -inf has no part; where a row sees no other one, the quotient is 0 / 0, not that of no key."""
    rng = np.random.default_rng([52, d, room])
    keys, offsets = [1, 40, 0, 33, 1500 if room > 1500 else 60], [0, 1, 2, 3, 5, 6]
    cache = Cache(rng, keys, 2, d, 16, BF16)
    k = cache.k[0].logical()
    gone = [[0], [3, 39], [], range(33), range(keys[4])]
    for b, js in enumerate(gone):
        for j in js:
            k[cache.table[b, j // 16], :, j % 16] = -np.inf
    cache.k[0] = HT.from_logical(k, BF16)
    widened(cache, room)
    q = HT.from_logical(0.1 + np.abs(rng.standard_normal([6, 4, d])), BF16)
    got, _ = run_paged(ctx, cache, keys, q, offsets)
    assert np.isnan(got[0]).all() and np.isnan(got[3:]).all() and not got[2].any()
    left = np.delete(np.arange(40), gone[1])
    ref, far = attend(q.logical()[1:2].astype(np.float64), cache.rows("k", 1)[left], cache.rows("v", 1)[left], [38], BF16)
    check(got[1:2], ref, far)
    # the same through packed rows
    k, v = (rows_of(rng, [sum(keys), 2, d], BF16) for _ in "kv")
    kl, at = k.logical(), np.concatenate([[0], np.cumsum(keys)])
    for b, js in enumerate(gone):
        kl[[at[b] + j for j in js]] = -np.inf
    got, _ = run_packed(ctx, q, HT.from_logical(kl, BF16), v, offsets, True, kv_offsets=at)
    assert np.isnan(got[0]).all() and np.isnan(got[3:]).all() and not got[2].any()
    ref, far = attend(q.logical()[1:2].astype(np.float64), kl[1:41][left], v.logical()[1:41][left].astype(np.float64), [38], BF16)
    check(got[1:2], ref, far)


# ---- layouts on the tuned kernel ----------------------------------------------------
@pytest.mark.parametrize("d,group", [(64, 0), (128, 0), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("order,page,dtype", [((0, 2, 1, 3), 16, BF16), ((1, 0, 2, 3), 32, capi.HALF), ((2, 1, 0, 3), 48, BF16)])
@pytest.mark.parametrize("keys,room", [([90, 1, 400], 0), ([90, 1, 2100], 4096)])
def test_paged_layouts(ctx, d, group, causal, order, page, dtype, keys, room):
    """Any order of a pool's dims, heads of Q outermost, rows of O apart, a scale, rows in front of the first sequence and
    behind the last, in one workgroup for each tile and cut into pieces."""
    rng = np.random.default_rng([53, d, group, page])
    cache = widened(Cache(rng, keys, 2, d, page, dtype, group, order=order), room)
    offsets = [2, 5, 6, 8]
    q = rows_of(rng, [11, 6, d], dtype, "heads")
    got, level = run_paged(ctx, cache, keys, q, offsets, causal, scale=0.11, o_how="wide")
    assert level == 2 and ctx.last_kernel().startswith(f"sdpa_paged d={d} bits={4 if group else 16} group={group} cut={int(room > 0)}")
    check_paged(cache, keys, q, offsets, got, causal, scale=0.11)


# ---- scales -------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale,tuned", [(1e4, True), (1e9, False), (1e30, False)])
def test_scales_that_leave_one_key(ctx, d, scale, tuned):
    """Scores that differ by at least 1: the largest one has all of the probability, whatever a chunk's other rows see.  It
    is rounded to bf16, and so is the result."""
    rng = np.random.default_rng([54, d])
    keys, lens = [70, 0, 33, 1100], [40, 2, 33, 3]
    offsets = np.concatenate([[0], np.cumsum(lens)])
    cache = widened(Cache(rng, keys, 1, d, 16, BF16), 2048)
    kl = np.zeros(cache.k[0].logical().shape, np.float32)
    for b, n in enumerate(keys):
        j = np.arange(n)
        order = rng.permutation(n)
        kl[cache.table[b, j // 16], 0, j % 16, 0], kl[cache.table[b, j // 16], 0, j % 16, 1] = order // 128, order % 128
    cache.k[0] = HT.from_logical(kl, BF16)
    ql = np.zeros([offsets[-1], 2, d])
    ql[:, :, 0], ql[:, :, 1] = 128, 1  # (q . k is the key's number in the permutation)
    q = HT.from_logical(ql, BF16)
    got, level = run_paged(ctx, cache, keys, q, offsets, scale=scale)
    assert level == (2 if tuned else 1)
    at = np.concatenate([[0], np.cumsum(keys)])
    k, v = (HT.from_logical(np.concatenate([cache.rows(x, b) for b in range(4)]), BF16) for x in "kv")
    packed, _ = run_packed(ctx, q, k, v, offsets, True, kv_offsets=at, scale=scale)
    for b, (n, m) in enumerate(zip(lens, keys)):
        score = k.logical()[at[b]:at[b + 1], 0, :2] @ [128, 1]
        for i in range(n):
            seen = max(m - n + i + 1, 0)
            want = v.logical()[at[b] + np.argmax(score[:seen]), 0] if seen else np.zeros(d)
            for out in (got, packed):
                check(out[offsets[b] + i], np.broadcast_to(want, [2, d]), np.abs(want) * 2.01 * 2.0 ** -8, f"{b} {i}")


# ---- strides of dims of one -----------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("stride", [0, 3, 8, 1 << 40])
def test_one_row_of_any_stride(ctx, d, stride):
    """The strides of dims of 1 are not used: neither their alignment nor their size matters, and what lies a stride behind
    the row is not taken for another one."""
    rng = np.random.default_rng([55, d])
    v = rng.standard_normal([1, 1, d])
    v[0, 0, d - 9] = np.inf
    q, k, v = HT.from_logical(rng.standard_normal([1, 4, d]), BF16), rows_of(rng, [1, 1, d], BF16), HT.from_logical(v, BF16)
    o = HT.from_logical(np.full([1, 4, d], 77.0), BF16)
    p = capi.SdpaPackedDesc()
    p.q, p.o = (capi.TensorDesc.make([1, 4, d], [stride, d, 1], BF16) for _ in "qo")
    p.k, p.v = (capi.TensorDesc.make([1, 1, d], [stride, stride, 1], BF16) for _ in "kv")
    p.batch, p.is_causal = 1, 1
    bufs, bo = [x.upload(ctx) for x in (q, k, v)], o.upload(ctx)
    assert ctx.lib.fhip_sdpa_packed_fwd_supported(p) == (1 if d == 80 else 2)
    ctx.sdpa_packed_fwd(p, *bufs, ints(ctx, [0, 1]), bo)
    assert np.array_equal(o.fetch(ctx, bo).logical(), np.broadcast_to(v.logical(), [1, 4, d]))
    cache = Cache(rng, [7], 1, d, 16, BF16)
    a = capi.CacheAppendDesc()
    a.q, a.q_out, a.k, a.v, a.cache = p.q, p.o, p.k, p.v, cache.desc()
    at = cache.upload(ctx)
    ctx.cache_append(a, at, bufs[1], bufs[2], ints(ctx, [0, 1]), q=bufs[0], q_out=bo)
    cache.fetch(ctx)
    assert np.array_equal(o.fetch(ctx, bo).logical(), q.logical()) and np.array_equal(cache.rows("v", 0)[6], v.logical()[0])
    r = capi.CacheReadDesc()
    r.k, r.v, r.cache = p.k, p.v, cache.desc()
    back = [HT.from_logical(np.full([1, 1, d], 77.0), BF16) for _ in "kv"]
    outs = [x.upload(ctx) for x in back]
    ctx.cache_read(r, at, ints(ctx, [0, 1]), *outs)
    assert np.array_equal(back[1].fetch(ctx, outs[1]).logical(), v.logical())
    g = capi.SdpaPagedDesc()
    g.q, g.o, g.cache, g.is_causal = p.q, p.o, cache.desc(), 0
    cache.v[0] = HT.from_logical(rng.standard_normal(cache.v[0].dims), BF16)
    ctx.sdpa_paged_fwd(g, cache.upload(ctx), bufs[0], ints(ctx, [0, 1]), bo)
    check_paged(cache, [7], q, [0, 1], o.fetch(ctx, bo).logical(), causal=False)


# ---- long lines of pieces -------------------------------------------------------------
@pytest.mark.parametrize("d,group,dtype", [(64, 0, BF16), (64, 64, capi.HALF)])
@pytest.mark.parametrize("what", ["many rows", "few rows"])
def test_long_lines(ctx, d, group, dtype, what):
    """Pieces of more than 64 chunks: their cuts move to the ends of segments that are near, and in 4 bits smaller ones follow
    the large ones.  Sequences from shorter than a move to longer than many pieces, joined by one team a row and by several."""
    rng = np.random.default_rng([56, d, group])
    if what == "many rows":
        hq, hk = 16, 2
        keys, rows = [9000, 5, 120, 20000, 640, 3333, 1, 300, 14000, 7000, 250, 4444], [32, 3, 32, 31, 32, 32, 1, 17, 32, 32, 32, 30]
    else:
        hq, hk = 32, 2
        keys, rows = [9000, 58500, 40], [1, 14, 1]
    line = sum(-(-n // 32) * -(-r * (hq // hk) // 16) * hk for n, r in zip(keys, rows))
    assert line > 768 * 64 and (sum(rows) * hq <= 512) == (what == "few rows")
    cache = Cache(rng, keys, hk, d, 64, dtype, group)
    offsets = np.concatenate([[0], np.cumsum(rows)])
    q = rows_of(rng, [sum(rows), hq, d], dtype)
    got, level = run_paged(ctx, cache, keys, q, offsets)
    assert level == 2 and ctx.last_kernel().endswith("cut=1")
    ql = q.logical().astype(np.float64)
    values = {x: cache.values(x) for x in "kv"}
    for b, (n, m) in enumerate(zip(rows, keys)):
        j = np.arange(m)
        k, v = (values[x][cache.table[b, j // 64], :, j % 64] for x in "kv")
        some = np.arange(n) if n < 16 else np.arange(b % 2, n, 2)  # (a row of each tile of 16: 2 positions of 8 heads)
        ref, far = attend(ql[offsets[b] + some], k, v, np.clip(m - n + 1 + some, 0, m), dtype, **steps_of(cache, b, m))
        check(got[offsets[b] + some], ref, far, f"sequence {b}")
    again, _ = run_paged(ctx, cache, keys, q, offsets)
    assert np.array_equal(got, again)


# ---- appended from odd addresses --------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, capi.HALF])
@pytest.mark.parametrize("group", [0, 32, 64])
def test_append_from_odd_addresses_stores_what_it_should(ctx, dtype, group):
    """The general kernel at the sizes of the vector one: both pools, codes and parameters, and nothing else of them."""
    rng = np.random.default_rng([57, group])
    keys, new, d = [30, 7], [3, 2], 64
    at = np.concatenate([[0], np.cumsum(new)])
    cache = Cache(rng, keys, 2, d, 16, dtype, group)
    before = [[t.logical() for t in x] for x in (cache.k, cache.v)]
    k, v = (rows_of(rng, [5, 2, d], dtype) for _ in "kv")
    bufs = [ctx.to_device(np.concatenate([np.zeros(1, x.storage.dtype), x.storage.reshape(-1)])) for x in (k, v)]
    a = capi.CacheAppendDesc()
    a.k, a.v, a.cache = k.desc(), v.desc(), cache.desc()
    ctx.cache_append(a, cache.upload(ctx), *(b.ptr + 2 for b in bufs), ints(ctx, at))
    assert ctx.last_kernel() == "cache_append_rows"
    cache.fetch(ctx)
    place = np.concatenate([np.arange(m - n, m) for n, m in zip(new, keys)])
    where = cache.table[np.repeat([0, 1], new), place // 16], place % 16
    check_held(cache, before[0], [t.logical() for t in cache.k], where, k.logical(), group, dtype, "K")
    check_held(cache, before[1], [t.logical() for t in cache.v], where, v.logical(), group, dtype, "V")


# ---- large pools, every step on one stream -----------------------------------------------
@pytest.mark.parametrize("group", [0, 64])
def test_a_pool_beyond_32_bits_on_one_stream(group):
    """test_serving_paths_gpu's steps with torch's current stream not the null one, of which a context makes a stream of its
    own: the copies into the pools and the calls are in order."""
    with torch.cuda.stream(torch.cuda.Stream()):
        test_serving_paths_gpu.test_a_pool_beyond_32_bits(group)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("group", [32, 64])
def test_missing_pages_and_keys_behind_the_table_in_f16(ctx, group):
    """Rows that see them are NaN, the others of their tile and sequence are not, in the kernel that follows the products'
    size too."""
    rng = np.random.default_rng([59, group])
    keys, rows = [40, 600, 20], [1, 300, 1]
    cache = widened(Cache(rng, keys, 1, 64, 16, capi.HALF, group), 2048)
    cache.table[1, 30] = cache.pool + 5  # (keys 480 .. 495)
    lengths = [40, 600, 2049]
    cache.table[2, :] = cache.table[0, 0]
    q = rows_of(rng, [302, 2, 64], capi.HALF)
    offsets = [0, 1, 301, 302]
    got, level = run_paged(ctx, cache, lengths, q, offsets)
    assert level == 2 and np.isnan(got[301]).all()
    seen = 301 + np.arange(300)
    assert np.isnan(got[1:301][seen > 480]).all() and np.isfinite(got[1:301][seen <= 480]).all()
    ql = q.logical().astype(np.float64)
    ref, far = attend(ql[:1], cache.rows("k", 0), cache.rows("v", 0), [40], capi.HALF, **steps_of(cache, 0, 40))
    check(got[:1], ref, far)
    cache.table[1, 30] = 0
    ref, far = attend(ql[1:181], cache.rows("k", 1, 480), cache.rows("v", 1, 480), seen[:180], capi.HALF, **steps_of(cache, 1, 480))
    check(got[1:181], ref, far)


@pytest.mark.parametrize("d,group", [(64, 0), (128, 0), (128, 64), (80, 0)])
@pytest.mark.parametrize("dtype", [BF16, capi.HALF])
@pytest.mark.parametrize("room", [0, 2048])
def test_rows_without_keys_beside_values_that_are_no_numbers(ctx, d, group, dtype, room):
    """More rows than keys, whose values are NaN or infinite: the first rows see none of them and are 0."""
    rng = np.random.default_rng([60, d, group])
    keys, rows = [2, 30, 1200 if room else 70], [5, 41, 3]
    offsets = np.concatenate([[0], np.cumsum(rows)])
    cache = widened(Cache(rng, keys, 1, d, 16, dtype, group), room)
    pool = cache.v[-1].logical()  # (values, or in 4 bits their parameters)
    for b in range(2):
        pool[cache.table[b, 0]] = np.nan if b else np.inf
    cache.v[-1] = HT.from_logical(pool, cache.v[-1].dtype)
    q = rows_of(rng, [offsets[-1], 2, d], dtype)
    got, _ = run_paged(ctx, cache, keys, q, offsets)
    assert not got[:3].any() and not got[5:16].any()
    assert not np.isfinite(got[3:5]).any() and not np.isfinite(got[16:46]).any()
    j = np.arange(keys[2])
    with np.errstate(invalid="ignore"):
        k, v = (cache.values(x)[cache.table[2, j // 16], :, j % 16] for x in "kv")
    ref, far = attend(q.logical()[46:].astype(np.float64), k, v, keys[2] - 2 + np.arange(3), dtype, **steps_of(cache, 2, keys[2]))
    check(got[46:], ref, far)
    if not group:
        at = np.concatenate([[0], np.cumsum(keys)])
        kp, vp = (HT.from_logical(np.concatenate([cache.rows(x, b) for b in range(3)]), dtype) for x in "kv")
        got, _ = run_packed(ctx, q, kp, vp, offsets, True, kv_offsets=at)
        assert not got[:3].any() and not got[5:16].any() and not np.isfinite(got[16:46]).any()
