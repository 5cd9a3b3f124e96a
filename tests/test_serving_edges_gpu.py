"""Packed sequences and paged caches at their edges: metadata of any value, sizes at the limit of a launch, long
lines of pieces, small and infinite values."""
import numpy as np
import pytest

from fusilli_amd import capi
from helpers import HT
from serving import Cache, attend, check
from test_serving_gpu import ints, rows_of

pytestmark = pytest.mark.gpu
BF16 = capi.BFLOAT16
INT_MIN = -2 ** 31


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
    cache = Cache(rng, keys, 2, d, 16, BF16)
    if room > cache.table.shape[1] * 16:
        cache.table = np.concatenate([cache.table, np.full([batch, room // 16 - cache.table.shape[1]], -7, np.int32)], 1)
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
