"""Rows in 8-bit codes, their products and tokens from logits for tests: the operators' formulas in 64 bits (in
f32 steps where the formula says so), and the bounds that their roundings allow."""
from __future__ import annotations

import numpy as np
import torch  # noqa: F401 (before the library, which then shares its runtime)

from fusilli_amd import capi

HALF_STEP = {capi.BFLOAT16: 2.0 ** -8, capi.HALF: 2.0 ** -11, capi.FLOAT: 2.0 ** -24}
UNIT = 2.0 ** -24


def matrix(shape, dtype, strides=None):
    return capi.TensorDesc.make(shape, strides or [shape[1], 1], dtype)


def guarded(ctx, host, before=0, behind=64):
    """`host`'s bytes on the device between guards: (buffer, address, what() -> the bytes, asserting the guards)."""
    raw = np.ascontiguousarray(host).view(np.uint8).reshape(-1)
    whole = np.concatenate([np.full(64 + before, 0xA5, np.uint8), raw, np.full(behind, 0xA5, np.uint8)])
    buf = ctx.to_device(whole)

    def what():
        got = buf.download(np.uint8, whole.size)
        a, b = 64 + before, 64 + before + raw.size
        assert (got[:a] == 0xA5).all() and (got[b:] == 0xA5).all(), "written outside"
        return got[a:b].view(host.dtype).reshape(host.shape)
    return buf, buf.ptr + 64 + before, what


# ---- rows to codes --------------------------------------------------------------
def front(x, kind, weight=None, up=None, eps=1e-6):
    """(y, bound on its relative error in f32 steps) of rows x [rows, K], in f64."""
    x = np.asarray(x, np.float64)
    if kind == "RMSNORM":
        # the sum of K squares: a thread's own ones in a row (at least 64 threads share a row), then a tree; half of
        # its error is left under the root; mean, epsilon, root, quotient and two products round once each
        k = x.shape[1]
        y = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * (1.0 if weight is None else np.asarray(weight, np.float64))
        return y, ((k / 64 + 12) / 2 + 6) * UNIT
    if kind == "SWISH_GATE":
        # exp is good to 2 steps of 2^-23, the sum, the quotient (2 steps of 2^-23) and the product round once each
        with np.errstate(over="ignore", invalid="ignore"):
            return x / (1.0 + np.exp(-x)) * np.asarray(up, np.float64), 12 * UNIT
    return x, 0.0


def check_codes(q, scale, y, rel):
    """Codes q and scales of rows whose y is good to `rel`."""
    y, q = np.asarray(y, np.float64), np.asarray(q, np.float64)
    for r in range(y.shape[0]):
        most = np.abs(y[r]).max()
        if not np.isfinite(y[r]).all():
            assert np.isnan(scale[r]) and not q[r].any(), f"row {r}"
        elif most == 0:
            assert scale[r] == 0 and not q[r].any(), f"row {r}"
        else:
            assert abs(scale[r] - most / 127) <= (rel + UNIT) * most / 127 + 2.0 ** -149, f"row {r}: scale {scale[r]}"
            # (the largest has `rel` too; the factor 127 / a and the product round once each)
            off = np.abs(q[r] - y[r] * (127 / most)) - 0.5 - 127 * (2 * rel + 2 * UNIT)
            assert off.max() <= 0, f"row {r}: code {int(off.argmax())} off by {off.max() + 0.5}"
            assert np.abs(q[r]).max() == 127


def codes_in_f32(x):
    """Codes and scales by the header's formula in f32, which numpy rounds as the kernels do."""
    x = np.asarray(x, np.float32)
    most = np.abs(x).max(1, keepdims=True)
    wide = np.where(most < np.float32(2.0 ** -100), np.float32(2.0 ** 64), np.float32(1))
    with np.errstate(all="ignore"):
        by = np.where(most > 0, np.float32(127) / (most * wide), np.float32(0)).astype(np.float32)
        q = np.clip(np.rint((x * wide) * by), -127, 127).astype(np.int8)
    return q, (most / np.float32(127))[:, 0]


# ---- products --------------------------------------------------------------------
def product(a, b, a_scale, b_scale, bias=None):
    """(C, bound on its error before its type) in f64."""
    total = a.astype(np.int64) @ b.astype(np.int64)
    assert np.abs(total).max(initial=0) < 2 ** 31
    c = total * np.asarray(a_scale, np.float64)[:, None] * np.asarray(b_scale, np.float64)[None]
    # the sum, its first product, the second with the bias: a rounding each
    bound = 2 * UNIT * np.abs(c) * 1.001
    if bias is not None:
        c = c + np.asarray(bias, np.float64)[None]
    return c, bound + UNIT * np.abs(c) * 1.001 + 2.0 ** -149


def check_product(got, c, bound, dtype):
    got = np.asarray(got, np.float64)
    least = {capi.BFLOAT16: 2.0 ** -133, capi.HALF: 2.0 ** -24, capi.FLOAT: 2.0 ** -149}[dtype]
    room = bound + HALF_STEP[dtype] * np.abs(c) * (1 + 2 * UNIT) + least
    if dtype == capi.HALF:  # (beyond its range: infinity)
        large = np.abs(c) > 65000
        got, c, room = np.where(large, 0, got), np.where(large, 0, c), np.where(large, 0, room)
    nan = np.isnan(c)
    assert np.array_equal(nan, np.isnan(got))
    off = np.where(nan, 0, np.abs(np.where(nan, 0, got - c)) - room)
    assert off.max(initial=-1) <= 0, f"{np.unravel_index(off.argmax(), off.shape)}: {off.max()} beyond the bound, {np.mean(off > 0):.2%}"


# ---- tokens ------------------------------------------------------------------------
def token(logits, u, t=1.0, k=0, p=1.0, least=0.0):
    """(token, probability) of one row, by the header's words."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l) + 0.0
    order = np.lexsort((np.arange(l.size), -l))
    order = order[l[order] > -np.inf]
    if order.size == 0:
        return -1, 0.0
    if not t > 0:
        return int(order[0]), 1.0
    s, most = l[order], l[order[0]]
    with np.errstate(all="ignore"):
        weight = np.where(s == most, 1.0, np.exp((s - most) / np.float64(np.float32(t))))
    held = [int(w) for w in np.rint(weight * 2.0 ** 40)]
    n = k if 0 < k < len(held) else len(held)
    total = sum(held[:n])
    if p < 1:
        need, run, m = float(np.float32(p)) * total, 0, 0
        while m < n and (m == 0 or run < need):
            run, m = run + held[m], m + 1
        n = m
    if least > 0:
        n = max(1, min(n, int((weight >= np.float64(np.float32(least))).sum())))
    total = sum(held[:n])
    at, run = float(np.float32(u)) * total if u > 0 else 0.0, 0
    for i in range(n):
        run += held[i]
        if run > at:
            return int(order[i]), held[i] / total
    last = max(i for i in range(n) if held[i])
    return int(order[last]), held[last] / total


def tokens(logits, uniform, t, k, p, least):
    got = [token(l, *s) for l, *s in zip(logits, uniform, t, k, p, least)]
    return np.array([g[0] for g in got]), np.array([g[1] for g in got])
