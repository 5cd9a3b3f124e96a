"""Tokens from logits for tests: the header's words in whole numbers, exactly as many bits as the operator keeps."""
from __future__ import annotations

import numpy as np


def weight_bits(words):
    """A weight of 1 is two to this: at most 46, and few enough that a row's sum stays within 2^62."""
    bits = 0
    while bits < 46 and words << (bits + 1) <= 1 << 62:
        bits += 1
    return bits


def draw(logits, u, t=1.0, k=0, p=1.0, least=0.0):
    """(token, probability) of one row.  Settings count as the f32 numbers that they are."""
    l = np.asarray(logits, np.float64)
    words = l.size
    l = np.where(np.isnan(l), -np.inf, l) + 0.0
    order = np.lexsort((np.arange(words), -l))
    order = order[l[order] > -np.inf]
    u, t, p, least = (float(np.float32(v)) for v in (u, t, p, least))
    if order.size == 0:
        return -1, 0.0
    if not t > 0:
        return int(order[0]), 1.0
    s = l[order]
    with np.errstate(all="ignore"):
        weight = np.where(s == s[0], 1.0, np.exp((s - s[0]) / t))
    one = 1 << weight_bits(words)
    run = np.cumsum(np.rint(weight * one).astype(np.int64))
    n = int(k) if 0 < k < s.size else s.size
    if p < 1:
        total = int(run[n - 1])
        need = min(max(1, int(np.ceil(p * float(total)))), total)
        n = int(np.searchsorted(run[:n], need, side="left")) + 1
    if least > 0:
        n = max(1, min(n, int((weight >= min(least, 1.0)).sum())))
        n = 1 if least > 1 else n
    kept = int(run[n - 1])
    # (u is 24 bits: below 1 the product is as far from `kept` as its 53 can tell)
    below = kept - 1 if u >= 1 else int(np.floor(u * float(kept))) if u > 0 else 0
    at = int(np.searchsorted(run[:n], below, side="right"))
    return int(order[at]), (int(run[at]) - (int(run[at - 1]) if at else 0)) / kept


def draws(logits, uniform, t, k, p, least):
    got = [draw(l, *s) for l, *s in zip(logits, uniform, t, k, p, least)]
    return np.array([g[0] for g in got]), np.array([g[1] for g in got])
