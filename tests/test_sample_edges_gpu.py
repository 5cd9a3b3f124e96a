"""Tokens from logits where the weights and the settings end, against the formula in whole numbers."""
import numpy as np
import pytest
import torch  # noqa: F401 (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
from quantized import guarded
from sampling import draws, weight_bits

pytestmark = pytest.mark.gpu
F32 = capi.FLOAT
# a wavefront, 256 and 1024 threads a row, parts of a row; and the kernel for any strides
PATHS = [(2, 1), (700, 1), (3000, 1), (18000, 1), (40000, 1), (700, 2), (40000, 2)]
JUST_BELOW_ONE = float(np.float32(1) - np.float32(2.0 ** -24))


def check(ctx, rows, uniform, t=1.0, k=0, p=1.0, least=0.0, stride=1):
    """rows: f32 values [rows, words]; the settings are one for all rows or one each."""
    n, words = np.shape(rows)
    x = HT.from_logical(np.asarray(rows, np.float32), F32, [stride * words, stride])
    each = lambda v, dt: np.ascontiguousarray(np.broadcast_to(np.asarray(v, dt), [n]))  # noqa: E731
    vec = dict(temperature=each(t, np.float32), top_k=each(k, np.int32), top_p=each(p, np.float32), min_p=each(least, np.float32))
    d = capi.SampleDesc()
    d.logits = x.desc()
    d.has_temperature = d.has_top_k = d.has_top_p = d.has_min_p = 1
    token, chance = guarded(ctx, np.full(n, -77, np.int32)), guarded(ctx, np.full(n, -7, np.float32))
    u = each(uniform, np.float32)
    ctx.sample(d, x.upload(ctx), ctx.to_device(u), token[1], probability=chance[1], **{i: ctx.to_device(v) for i, v in vec.items()})
    want, expected = draws(x.logical(), u, *vec.values())
    got = token[2]()
    assert np.array_equal(got, want), [(i, got[i], want[i], u[i], *(v[i] for v in vec.values())) for i in np.flatnonzero(got != want)][:5]
    # (a weight is a unit off at most where the exponential's last place is, and so is each of the sum's; one rounding)
    unit = 2.0 ** -weight_bits(words)
    assert (np.abs(chance[2]() - expected) <= 2.0 ** -24 * expected + unit * (1 + words * expected)).all()


@pytest.mark.parametrize("words,stride", PATHS)
def test_words_whose_weight_is_the_last_unit(ctx, words, stride):
    """exp(-32) is 0.89 of 2^-46 and counts as one: its word is drawn by numbers from 1 on, which count as the nearest
    below 1, and by none that the rows' other words leave out."""
    far = np.float32([31.5, 31.999998, 32.0, 32.000004, 32.00001, 32.00002, 32.00004, 32.3, 32.5, 32.7, 33.0, 33.00002, 40.0])
    rows = np.full([2 * len(far), words], -np.inf, np.float32)
    rows[::2, words - 1], rows[::2, 0] = 0, -far      # (0 ahead, behind it one word at each distance)
    rows[1::2, 0], rows[1::2, words - 1] = 16, 16 - far  # (both sides of 0)
    for u in (1.0, 1.5, np.inf, JUST_BELOW_ONE, 0.0, np.nan, -3.0):
        check(ctx, rows, u, stride=stride)
        check(ctx, rows, u, k=2, p=0.99999994, stride=stride)
    half = np.float32(np.where(np.isfinite(rows), rows / 2, rows))
    check(ctx, half, 1.0, t=0.5, stride=stride)
    check(ctx, half, 1.0, t=0.5, least=1e-14, stride=stride)


@pytest.mark.parametrize("words,stride", [(w, s) for w, s in PATHS if w > 2])
def test_many_words_at_the_last_unit(ctx, words, stride):
    """Hundreds of words on either side of 32 among ordinary ones: numbers from 1 on draw the last that weighs a unit."""
    rng = np.random.default_rng([1, words])
    rows = rng.normal(size=[6, words]).astype(np.float32) - 60
    for row in rows:
        at = rng.permutation(words)[:400]
        row[at[:200]] = -rng.uniform(31.9, 32.1, 200)
        row[at[200:300]] = np.float32(-32) - np.float32(2.0 ** -18) * rng.integers(0, 12, 100)
        row[at[300:398]] = rng.normal(size=98) - 8
        row[at[398]] = 0
    for u in (1.0, 2.0, JUST_BELOW_ONE, 0.5):
        check(ctx, rows, u, stride=stride)
    check(ctx, rows, 1.0, k=[0, 5, 150, 250, 390, 399], stride=stride)
    check(ctx, rows, 1.0, p=[1.0, 0.5, 0.9, 0.99999994, 1.0, 1.0], least=[0.0, 0.0, 0.0, 0.0, 1e-13, 1e-14], stride=stride)


@pytest.mark.parametrize("words,stride", [(w, s) for w, s in PATHS if w > 2])
@pytest.mark.parametrize("dtype_seed", [0, 1])
def test_numbers_beyond_their_range(ctx, words, stride, dtype_seed):
    """Ordinary rows with each setting: numbers from 1 on, infinite, negative and NaN, every row against the formula."""
    rng = np.random.default_rng([2, words, dtype_seed])
    n = 12
    rows = rng.normal(size=[n, words]) * rng.choice([0.5, 2.0, 6.0], [n, 1])
    t, k = rng.choice([0.0, 0.7, 1.0, 1.3], n), rng.choice([0, 1, 20, words // 3], n)
    p, least = rng.choice([1.0, 0.9, 0.5], n), rng.choice([0.0, 0.05, 1.0], n)
    for u in (1.0, 1.5, np.inf, -1.0, -np.inf, np.nan):
        check(ctx, rows, u, t, k, p, least, stride=stride)


COLD = PATHS[1:]


@pytest.mark.parametrize("words,stride", COLD)
@pytest.mark.parametrize("t", [1e-45, 1e-42, 1e-39, 2e-38, 1e-33, 1e-29, 8.07e-28, 8.08e-28, 1e-26])
def test_rows_that_are_nearly_greedy(ctx, words, stride, t):
    """Temperatures down to the smallest number above 0, with words a few of them apart and others beyond 64 of them."""
    rng = np.random.default_rng([3, words])
    t = float(np.float32(t))
    rows = np.full([8, words], -1.0, np.float32)
    for i, row in enumerate(rows):
        at = rng.permutation(words)[:200]
        row[at] = -np.float32(np.maximum(np.rint(rng.uniform(0, [5, 40, 200, 1000][i % 4], 200)), 0) * t)
        row[at[0]] = 0
        row[at[1]] = [-1e-30, -7e-36, -3e-36, -1e-37][i % 4]
        if i >= 4:  # (every word near the largest)
            row[:] = np.where(row == -1, np.float32(-0.25 * t), row)
    for u in (0.05, 0.4, 0.8, 0.99, 1.0):
        check(ctx, rows, u, t, stride=stride)
        check(ctx, rows, u, t, k=[0, 3, 50, 0, 0, 7, 0, 100], p=[0.9, 1.0, 0.5, 0.99, 0.9, 1.0, 0.5, 0.99],
              least=[0.0, 0.02, 0.0, 0.3, 0.02, 0.0, 0.99999994, 1.0], stride=stride)


@pytest.mark.parametrize("words,stride", COLD)
@pytest.mark.parametrize("apart", [1e-45, 1e-30, 1e-12, 1e-10, 1e-9, 1e-8, 1e-7, 1.0, 1e30])
def test_rows_of_infinite_temperature(ctx, words, stride, apart):
    """Every word weighs the same, however close together or far apart they are."""
    rng = np.random.default_rng([4, words])
    rows = (-rng.integers(0, 50, [4, words]) * np.float64(apart)).astype(np.float32)
    rows[1, ::3] = -np.inf
    rows[2, 1::2] = 0
    for u in (0.0, 0.3, 0.7, JUST_BELOW_ONE, 1.0):
        check(ctx, rows, u, np.inf, stride=stride)
        check(ctx, rows, u, np.inf, k=[0, 9, words // 2, 0], p=[0.5, 1.0, 0.9, 0.25], least=[0.0, 0.5, 1.0, 0.0], stride=stride)


@pytest.mark.parametrize("rows,words", [(2, 1 << 20), (2, (1 << 22) + 3), (1, 1 << 24)])
def test_large_vocabularies_of_distinct_logits(ctx, rows, words):
    """So many words in each bucket that those in question outnumber what a list holds: all of the row's words answer."""
    rows = np.random.default_rng([5, words]).normal(size=[rows, words]).astype(np.float32) * np.float32([[1.5], [3.0]][:rows])
    check(ctx, rows, [0.83, 0.4][:len(rows)], p=0.95)
    check(ctx, rows, [0.02, 0.99][:len(rows)], t=1.25, k=words // 3, p=0.9, least=[1e-6, 0.0][:len(rows)])
