"""Packed sequences and paged caches for tests: the operators' formulas in 64
bits, and the bounds that their roundings allow."""
from __future__ import annotations

import os
import subprocess
import tempfile

import numpy as np

from fusilli_amd import capi
from oracle import oracle
from helpers import HT

# half a step of a type, relative to the value
HALF_STEP = {capi.BFLOAT16: 2.0 ** -8, capi.HALF: 2.0 ** -11, capi.FLOAT: 2.0 ** -24}


def starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def rotation_table(places, rotary, base=10000.0):
    step = base ** (-np.arange(0, rotary, 2) / rotary)
    angle = np.arange(places)[:, None] * step
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def turn(x, table, pos, interleaved):
    """Rows [T, H, D] turned by row pos of the table, in f64."""
    y = np.array(x, np.float64)
    r = table.shape[1]
    cos, sin = (t[:, None].astype(np.float64) for t in np.split(table[pos], 2, axis=1))
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * cos - v * sin, v * cos + u * sin
    return y


def turn_bound(x, table, pos, interleaved, dtype):
    """|a cos| + |b sin| of every turned element: two products and their sum are rounded in f32, the
    result to its type."""
    t = np.abs(table)
    r = t.shape[1]
    cos, sin = (s[:, None].astype(np.float64) for s in np.split(t[pos], 2, axis=1))
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y = np.abs(np.array(x, np.float64))
    u, v = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * cos + v * sin, v * cos + u * sin
    return 3 * 2.0 ** -24 * y


def to_groups(x, group):
    """What 4 bits keep of x [..., D]: codes, scales and lows, by the header's formula in f32 steps
    (numpy rounds each to even as the kernels do)."""
    y = np.asarray(x, np.float32).reshape(*np.shape(x)[:-1], -1, group)
    with np.errstate(all="ignore"):
        low = y.min(-1, keepdims=True).astype(np.float16)
        wide = np.maximum(y.max(-1, keepdims=True) - low.astype(np.float32), np.float32(0))
        scale = (wide / np.float32(15)).astype(np.float16)
        bad = ~np.isfinite(y).all(-1, keepdims=True) | ~np.isfinite(low) | ~np.isfinite(scale)
        by = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0))
        code = np.clip(np.rint((y - low.astype(np.float32)) * by), 0, 15)
    code = np.where(bad, 0, code).astype(np.uint8).reshape(np.shape(x))
    scale, low = (np.where(bad, np.float16(np.nan), t)[..., 0] for t in (scale, low))
    return code, scale, low


def from_groups(code, scale, low):
    group = code.shape[-1] // scale.shape[-1]
    f = lambda t: np.repeat(t.astype(np.float64), group, -1)  # noqa: E731
    return f(low) + f(scale) * code


class Cache:
    """A paged cache on the host: pools, table and lengths; `order` says which dim of
    [pages, heads, page size, dim] lies outside which."""

    def __init__(self, rng, keys, heads, d, page, dtype, group=0, dv=None, order=(0, 1, 2, 3), fill=None, spare=3):
        self.keys, self.heads, self.d, self.dv, self.page, self.dtype, self.group = keys, heads, d, dv or d, page, dtype, group
        need = [max(1, -(-n // page)) for n in keys]
        self.pool = sum(need) + spare
        pages = rng.permutation(self.pool)
        self.table = np.full([len(keys), max(need) + 1], -7, np.int32)  # (entries behind the last page are never read)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = pages[at:at + n]
            at += n
        self.order = order
        self.k, self.v = (self._pool(rng, dim, fill) for dim in (self.d, self.dv))

    def _strides(self, dims):
        st, run = [0] * 4, 1
        for i in reversed(self.order):
            st[i] = run
            run *= dims[i]
        return st

    def _pool(self, rng, d, fill):
        x = rng.standard_normal([self.pool, self.heads, self.page, d]) if fill is None else \
            np.full([self.pool, self.heads, self.page, d], fill)
        if not self.group:
            return [HT.from_logical(x, self.dtype, self._strides(x.shape))]
        code, scale, low = to_groups(x, self.group)
        two = (code[..., ::2] | code[..., 1::2] << 4).astype(np.uint8)
        pair = np.stack([scale, low], -1).reshape(*scale.shape[:-1], -1)
        return [HT.from_logical(two.astype(np.float64), capi.UINT8, self._strides(two.shape)),
                HT(pair.shape, self._strides(pair.shape), capi.HALF, oracle.to_storage(pair.astype(np.float16), self._strides(pair.shape)))]

    def values(self, which):
        """What a pool holds, [pages, heads, page size, dim] in f64."""
        x = self.k if which == "k" else self.v
        if not self.group:
            return np.asarray(x[0].logical(), np.float64)
        two, pair = x[0].logical().astype(np.uint8), x[1].logical()
        code = np.stack([two & 15, two >> 4], -1).reshape(*two.shape[:-1], -1)
        return from_groups(code, pair[..., ::2], pair[..., 1::2])

    def rows(self, which, b, n=None):
        """The first n keys or values of sequence b, [n, heads, dim]."""
        j = np.arange(self.keys[b] if n is None else n)
        return self.values(which)[self.table[b, j // self.page], :, j % self.page]

    def upload(self, ctx, lengths=None):
        self.bufs = [[t.upload(ctx) for t in x] for x in (self.k, self.v)]
        self.bufs.append([ctx.to_device(self.table), ctx.to_device(np.asarray(self.keys if lengths is None else lengths, np.int32))])
        (k, *kp), (v, *vp), (table, lens) = self.bufs
        return capi.CachePointers.make(k, v, table, lens, *(kp + vp))

    def fetch(self, ctx):
        for x, bufs in zip((self.k, self.v), self.bufs):
            for t, buf in zip(x, bufs):
                t.fetch(ctx, buf)

    def desc(self):
        c = capi.CacheDesc()
        c.k, c.v = self.k[0].desc(), self.v[0].desc()
        if self.group:
            c.k_params, c.v_params = self.k[1].desc(), self.v[1].desc()
        c.batch, c.pages_per_sequence = self.table.shape
        c.page_stride = self.table.shape[1]
        return c


def attend(q, k, v, seen, dtype, scale=None, v_step=None, k_step=None):
    """Rows q [n, hq, d] over k, v [m, hkv, d]; row i sees the first seen[i] keys.  Returns the result
    in f64 and how far from it a kernel may be:

      * 16-bit kernels round each probability, off by u p at most: u sum(p |v|) / sum(p) (in 4 bits
        p times the scale is rounded: the codes at their most, v_step = 15 scales, count instead), and the result;
      * scores are sums of d products in f32, p errs with them by a factor 1 + 2 |ds|, and through
        the argument of exp2 by |s| 2^-22; sums over m keys are in f32.  In 4 bits the codes are
        multiplied as 128 + c: k_step (143 scales and the low values) in place of |k|.
    """
    n, hq, d = q.shape
    m, hkv = k.shape[:2]
    scale = 1 / np.sqrt(d) if scale is None else scale
    u, f = HALF_STEP[dtype], 2.0 ** -24
    out, far = np.zeros([n, hq, v.shape[2]]), np.zeros([n, hq, v.shape[2]])
    for h in range(hq):
        g = h * hkv // hq
        s = q[:, h] @ k[:, g].T * scale
        ds = np.abs(q[:, h]) @ (np.abs(k[:, g]) if k_step is None else k_step[:, g]).T * abs(scale) * (d + 4) * f
        for i in range(n):
            if seen[i] <= 0:
                continue
            si, vi = s[i, :seen[i]], v[:seen[i], g]
            p = np.exp(si - si.max())
            p /= p.sum()
            out[i, h] = p @ vi
            size = p @ np.abs(vi)
            step = size if v_step is None else p @ v_step[:seen[i], g]
            err = 2 * ds[i, :seen[i]] + np.abs(si - si.max()) * 4 * f
            # (a weighted mean: the error of p moves it by that of v against the mean)
            far[i, h] = ((err * p) @ np.abs(vi) + (err @ p) * size) * 1.1 + (seen[i] + 16) * f * 3 * (size + 10 * step)
            if dtype != capi.FLOAT:
                far[i, h] += u * step
            far[i, h] += u * np.abs(out[i, h]) * 1.01 + (2.0 ** -25 if dtype == capi.HALF else 0)
    return out, far


def check(got, ref, far, what=""):
    bad = ~(np.abs(got - ref) <= far)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(np.abs(got - ref) / far, nan=np.inf, posinf=1e30), -1)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside, worst at {at}: {got[at]} for {ref[at]} +- {far[at]}")


def cpp_binary(name, timeout, *only):
    """Runs a graph-API test binary, whose cache files go to a directory of this run."""
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", name)
    with tempfile.TemporaryDirectory(prefix="fusilli_cache_") as where:
        proc = subprocess.run([path, *only], capture_output=True, text=True, timeout=timeout,
                              env=dict(os.environ, FUSILLI_CACHE_DIR=where))
        left = [f for _, _, files in os.walk(where) for f in files]
    assert proc.returncode == 0 and "cases, 0 failed checks" in proc.stdout, proc.stdout[-4000:] + proc.stderr[-2000:]
    assert not left, left[:5]
    return proc.stdout
