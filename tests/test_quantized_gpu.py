"""Rows in 8-bit codes, products of codes and tokens from logits against their formulas in 64 bits, through the C ABI."""
import ctypes

import numpy as np
import pytest
import torch  # (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
from quantized import check_codes, check_product, codes_in_f32, front, guarded, product, tokens
from serving import cpp_binary

pytestmark = pytest.mark.gpu
BF16, F16, F32 = capi.BFLOAT16, capi.HALF, capi.FLOAT
TYPES = [BF16, F16, F32]
NAME = {BF16: "bf16", F16: "f16", F32: "f32"}


def rng_of(*seed):
    return np.random.default_rng(list(seed))


# ---- rows to codes ----------------------------------------------------------------
def quantize(ctx, x, kind="NONE", weight=None, up=None, eps=1e-6, q_strides=None, scale_stride=1, x_shift=0, q_shift=0):
    """x, up, weight: HT.  -> (codes, scales)"""
    rows, k = x.dims
    d = capi.QuantizeRowsDesc()
    d.x, d.front, d.epsilon = x.desc(), capi.QUANTIZE_FRONT[kind], eps
    q = HT.empty([rows, k], capi.INT8, q_strides, fill=77)
    d.q, d.scale_stride = q.desc(), scale_stride
    if weight is not None:
        d.has_weight, d.weight_dtype, d.weight_stride = 1, weight.dtype, weight.strides[0]
    if up is not None:
        d.up = up.desc()
    held = k <= 32768 and rows < 2 ** 21 and all(k == 1 or t.strides[-1] == 1 for t in (x, up, weight, q) if t is not None)
    assert ctx.lib.fhip_quantize_rows_supported(d) == (2 if held else 1)
    bx, px, _ = guarded(ctx, x.storage, x_shift)
    bu, pu, _ = guarded(ctx, up.storage, x_shift) if up is not None else (None, None, None)
    bw, pw, _ = guarded(ctx, weight.storage) if weight is not None else (None, None, None)
    bq, pq, codes = guarded(ctx, q.storage, q_shift)
    scales = np.full((rows - 1) * scale_stride + 1, -5.0, np.float32)
    bs, ps, scales_back = guarded(ctx, scales)
    ctx.quantize_rows(d, px, pq, ps, up=pu, weight=pw)
    assert ctx.last_kernel() == ("quantize_rows_held" if held else "quantize_rows_generic")
    q.storage = codes()
    touched = np.zeros(q.storage.size, bool)
    touched[(np.arange(rows)[:, None] * q.strides[0] + np.arange(k) * q.strides[1]).reshape(-1)] = True
    assert (q.storage[~touched] == 77).all()
    s = scales_back()
    assert (np.delete(s, np.arange(rows) * scale_stride) == -5.0).all()
    return q.logical().astype(np.int64), s[::scale_stride]


SIZES = [(1, 1), (1, 2048), (3, 7), (5, 1001), (17, 4096), (2, 16384), (2, 20008), (300, 96), (33, 8), (4, 5120),
         (2, 32768), (3, 32767), (2, 32769), (6, 511), (3, 513), (5, 8193)]


@pytest.mark.parametrize("kind", ["NONE", "RMSNORM", "SWISH_GATE"])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantize(ctx, kind, dtype, rows, k):
    rng = rng_of(1, rows, k, dtype)
    x = HT.from_logical(rng.normal(size=[rows, k]) * 2, dtype)
    weight = HT.from_logical(1 + 0.1 * rng.normal(size=[k]), dtype) if kind == "RMSNORM" else None
    up = HT.from_logical(rng.normal(size=[rows, k]), dtype) if kind == "SWISH_GATE" else None
    q, s = quantize(ctx, x, kind, weight, up)
    y, rel = front(x.logical(), kind, weight and weight.logical(), up and up.logical())
    check_codes(q, s, y, rel)
    if kind == "NONE":
        exact_q, exact_s = codes_in_f32(x.logical())
        assert np.array_equal(q, exact_q) and np.array_equal(s, exact_s)


@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("strides", ["padded", "columns", "every_second", "odd_address", "one_row_for_all"])
def test_quantize_strides(ctx, dtype, strides):
    rows, k = 9, 264
    rng = rng_of(2, dtype)
    x_strides = {"padded": [k + 13, 1], "columns": [1, rows], "every_second": [2 * k, 2], "odd_address": None,
                 "one_row_for_all": [0, 1]}[strides]
    values = rng.normal(size=[rows, k])
    if strides == "one_row_for_all":
        values[:] = values[:1]
    x = HT.from_logical(values, dtype, x_strides)
    up = HT.from_logical(rng.normal(size=[rows, k]), dtype, [k + 5, 1])
    q_strides = {"padded": [k + 3, 1], "columns": [1, rows], "every_second": [2 * k, 2], "odd_address": None,
                 "one_row_for_all": [k + 8, 1]}[strides]
    shift = 0 if strides != "odd_address" else capi.DTYPE_SIZE[dtype]
    for kind in ("NONE", "SWISH_GATE", "RMSNORM"):
        q, s = quantize(ctx, x, kind, up=up if kind == "SWISH_GATE" else None, q_strides=q_strides, scale_stride=3,
                        x_shift=shift, q_shift=1 if shift else 0)
        check_codes(q, s, *front(x.logical(), kind, up=up.logical()))


@pytest.mark.parametrize("k", [40, 1000, 4096])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_quantize_odd_rows(ctx, dtype, k):
    """Zeros, infinities, NaN, subnormals and one large value among small ones."""
    x = rng_of(3, k).normal(size=[12, k])
    x[0] = 0
    x[1, k // 2] = np.inf
    x[2, 0] = -np.inf
    x[3, k - 1] = np.nan
    x[4] *= 1e-30 if dtype != F16 else 1e-6
    x[5] = -0.0
    x[6, 1:] = 0
    x[7] *= 2.0 ** -128 if dtype != F16 else 2.0 ** -23
    x[8, 3] = 6e4
    x[9] = 3.0e38 if dtype != F16 else 65504
    x[10, :] = -1.0
    x = HT.from_logical(x, dtype)
    q, s = quantize(ctx, x)
    with np.errstate(all="ignore"):
        exact_q, exact_s = codes_in_f32(x.logical())
    bad = ~np.isfinite(x.logical()).all(1)
    assert np.array_equal(bad, np.isnan(s)) and not q[bad].any()
    assert np.array_equal(q[~bad], exact_q[~bad]) and np.array_equal(s[~bad], exact_s[~bad])


@pytest.mark.parametrize("front_kind", ["RMSNORM", "SWISH_GATE"])
def test_quantize_odd_rows_behind_a_front(ctx, front_kind):
    rng = rng_of(4)
    x = rng.normal(size=[8, 512])
    x[0] = 0
    x[1, 5] = np.nan
    x[2, 7] = np.inf
    x[3] *= 1e-12
    x[4] = -200.0
    x[5, 100] = 1e18
    x = HT.from_logical(x, BF16)
    up = HT.from_logical(rng.normal(size=[8, 512]), BF16) if front_kind == "SWISH_GATE" else None
    q, s = quantize(ctx, x, front_kind, up=up)
    with np.errstate(all="ignore"):
        y, rel = front(x.logical(), front_kind, up=up and up.logical())
    keep = [0, 3, 5, 6, 7] + ([2] if front_kind == "SWISH_GATE" else [])
    if front_kind == "SWISH_GATE":  # (exp(-200) is 0 in f32; in 64 bits the row is 1e-85)
        assert s[4] == 0 and not q[4].any()
    else:
        keep.append(4)
        assert np.isnan(s[2])
    check_codes(q[keep], s[keep], y[keep], rel)
    assert np.isnan(s[1]) and not q[1].any()


def test_quantize_weight_of_another_type_and_stride(ctx):
    rng = rng_of(5)
    x = HT.from_logical(rng.normal(size=[6, 768]), BF16)
    for weight in (HT.from_logical(rng.normal(size=[768]), F32), HT.from_logical(rng.normal(size=[768]), F16),
                   HT.from_logical(rng.normal(size=[768]), BF16, [3]), None):
        q, s = quantize(ctx, x, "RMSNORM", weight, eps=1e-3)
        check_codes(q, s, *front(x.logical(), "RMSNORM", weight and weight.logical(), eps=1e-3))


@pytest.mark.parametrize("k", [96, 1024, 40000])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=NAME.get)
def test_quantize_squares_beyond_f32(ctx, dtype, k):
    """A row of finite numbers whose squares' sum is infinite has no scale, rather than codes of zeros."""
    x = np.ones([3, k])
    x[1, k // 3] = 1e25
    q, s = quantize(ctx, HT.from_logical(x, dtype), "RMSNORM")
    assert np.isnan(s[1]) and not q[1].any()
    assert (q[[0, 2]] == 127).all() and np.isfinite(s[[0, 2]]).all()


@pytest.mark.parametrize("k", [96, 1024, 40000])
def test_quantize_gate_of_large_numbers(ctx, k):
    """x / (1 + exp(-x)) where exp leaves f32's range: nearly x, or nearly nothing."""
    x = rng_of(6, k).normal(size=[6, k])
    x[0] = 1e30
    x[1] = np.linspace(-95, -85, k)  # (a row of the smallest results: scales stay normal numbers)
    x[2] = np.where(np.arange(k) % 2, -3e38, 3e38)
    x[3, 1] = -np.inf
    x[4] = np.linspace(-150, 150, k)
    x = HT.from_logical(x, F32)
    up = HT.from_logical(np.where(np.arange(k) % 3, 1.0, -0.5)[None].repeat(6, 0), F32)
    q, s = quantize(ctx, x, "SWISH_GATE", up=up)
    y, rel = front(x.logical(), "SWISH_GATE", up=up.logical())
    keep = [0, 1, 2, 4, 5]
    check_codes(q[keep], s[keep], y[keep], rel)
    assert np.isnan(s[3]) and not q[3].any()


# ---- products ------------------------------------------------------------------------
def multiply(ctx, a, b, a_scale, b_scale, dtype=BF16, bias=None, a_strides=None, b_strides=None, o_strides=None,
             epilogue=(), c_dtype=None, shift=0, fast=None, a_stride=1, b_stride=1):
    """a, b: codes; scales and bias: vectors (HT bias).  epilogue: (op, HT or None) each.  -> OUT's values"""
    (m, k), n = a.shape, b.shape[1]
    d = capi.MatmulQuantizedDesc()
    ha, hb = HT.from_logical(a, capi.INT8, a_strides), HT.from_logical(b, capi.INT8, b_strides)
    out = HT.empty([m, n], dtype, o_strides, fill=3)
    d.a, d.b, d.out, d.out_dtype = ha.desc(), hb.desc(), out.desc(), dtype
    d.c = capi.TensorDesc.make([m, n], [n, 1], c_dtype or dtype)
    d.a_scale_stride, d.b_scale_stride = a_stride, b_stride
    if bias is not None:
        d.has_bias, d.bias_dtype, d.bias_stride = 1, bias.dtype, bias.strides[0]
    d.epilogue = capi.make_epilogue([e for e, _ in epilogue])
    supported = ctx.lib.fhip_matmul_quantized_supported(d)
    assert supported == (2 if fast else supported if fast is None else 1)
    keep = [guarded(ctx, ha.storage, shift), guarded(ctx, hb.storage, shift),
            guarded(ctx, np.repeat(np.asarray(a_scale, np.float32), max(a_stride, 1))),
            guarded(ctx, np.repeat(np.asarray(b_scale, np.float32), max(b_stride, 1))),
            guarded(ctx, bias.storage) if bias is not None else (None, None, None)]
    operands = [guarded(ctx, x.storage) for _, x in epilogue if x is not None]
    o = guarded(ctx, out.storage)
    ctx.matmul_quantized(d, *[x[1] for x in keep[:4]], o[1], bias=keep[4][1], epilogue_operands=[x[1] for x in operands])
    out.storage = o[2]()
    touched = np.zeros(out.storage.size, bool)
    touched[(np.arange(m)[:, None] * out.strides[0] + np.arange(n) * out.strides[1]).reshape(-1)] = True
    assert (out.storage[~touched] == 3).all()
    return out.logical()


def codes(rng, *shape):
    return np.clip(np.rint(rng.normal(size=shape) * 40), -128, 127).astype(np.int8)


def scales(rng, n):
    return (0.01 + 0.05 * rng.random(n)).astype(np.float32)


MNK = [(1, 1, 1), (1, 64, 16), (1, 4096, 4096), (2, 100, 17), (5, 1000, 333), (16, 128, 64), (33, 65, 1001), (64, 512, 2048),
       (127, 129, 128), (128, 128, 128), (200, 384, 1040), (256, 256, 512), (300, 520, 656), (512, 640, 4096), (777, 1400, 1000),
       (1000, 24, 64), (3, 3000, 5), (130, 4096, 15), (1025, 257, 256)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("m,n,k", MNK)
def test_product(ctx, dtype, m, n, k):
    rng = rng_of(6, m, n, k)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m), scales(rng, n)
    bias = HT.from_logical(rng.normal(size=[n]), dtype) if (m + n) % 2 else None
    got = multiply(ctx, a, b, sa, sb, dtype, bias, b_strides=[1, k])
    check_product(got, *product(a, b, sa, sb, bias and bias.logical()), dtype)


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (7, 48, 100), (130, 300, 257), (256, 512, 384), (300, 260, 1024)])
@pytest.mark.parametrize("a_along,b_along", [(1, 1), (1, 0), (0, 1), (0, 0)])
@pytest.mark.parametrize("pad", [0, 1, 16])
def test_product_orders(ctx, m, n, k, a_along, b_along, pad):
    rng = rng_of(7, m, n, k)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m), scales(rng, n)
    got = multiply(ctx, a, b, sa, sb, BF16, a_strides=[k + pad, 1] if a_along else [1, m + pad],
                   b_strides=[1, k + pad] if b_along else [n + pad, 1], o_strides=[n + pad, 1], shift=pad % 16)
    check_product(got, *product(a, b, sa, sb), BF16)


@pytest.mark.parametrize("m,n,k", [(5, 40, 64), (150, 200, 256), (256, 256, 256)])
@pytest.mark.parametrize("layout", ["out_columns", "out_every_second", "operands_every_second"])
def test_product_strides(ctx, m, n, k, layout):
    rng = rng_of(8, m, n)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m), scales(rng, n)
    kw = {"out_columns": dict(o_strides=[1, m + 3]), "out_every_second": dict(o_strides=[2 * n, 2]),
          "operands_every_second": dict(a_strides=[2 * k, 2], b_strides=[2, 2 * k])}[layout]
    check_product(multiply(ctx, a, b, sa, sb, F16, **kw), *product(a, b, sa, sb), F16)


@pytest.mark.parametrize("m,n,k", [(3, 50, 48), (130, 140, 256), (256, 384, 512)])
def test_product_one_scale_and_strides_between(ctx, m, n, k):
    rng = rng_of(9, m)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m), scales(rng, n)
    got = multiply(ctx, a, b, sa[:1], sb, F32, a_stride=0)
    check_product(got, *product(a, b, np.repeat(sa[:1], m), sb), F32)
    got = multiply(ctx, a, b, sa, sb[:1], F32, b_stride=0)
    check_product(got, *product(a, b, sa, np.repeat(sb[:1], n)), F32)
    bias = HT.from_logical(rng.normal(size=[n]), F16, [4])
    got = multiply(ctx, a, b, sa, sb, F32, bias, a_stride=2, b_stride=5)
    check_product(got, *product(a, b, sa, sb, bias.logical()), F32)


@pytest.mark.parametrize("bias_dtype", TYPES, ids=NAME.get)
def test_product_bias_types(ctx, bias_dtype):
    rng = rng_of(10)
    a, b, sa, sb = codes(rng, 140, 256), codes(rng, 256, 272), scales(rng, 140), scales(rng, 272)
    bias = HT.from_logical(rng.normal(size=[272]) * 100, bias_dtype)
    for dtype in TYPES:
        check_product(multiply(ctx, a, b, sa, sb, dtype, bias), *product(a, b, sa, sb, bias.logical()), dtype)


@pytest.mark.parametrize("m,n,k", [(1, 128, 131071), (1, 130, 131071), (160, 144, 131056)])
def test_product_largest_sums(ctx, m, n, k):
    """-128 times -128 all along the longest K."""
    a, b = np.full([m, k], -128, np.int8), np.full([k, n], -128, np.int8)
    b[:, 1] = 127
    one = np.ones(max(m, n), np.float32)
    got = multiply(ctx, a, b, one[:m], one[:n], F32, b_strides=[1, k])
    total = np.full([m, n], k * 16384.0)
    total[:, 1] = -128.0 * 127 * k
    check_product(got, total, 2.0 ** -24 * np.abs(total), F32)


@pytest.mark.parametrize("m,n,k", [(4, 40, 64), (130, 260, 256), (300, 512, 512)])
def test_product_scales_that_are_no_numbers(ctx, m, n, k):
    """A row or column whose scale is NaN or infinite shows there and nowhere else."""
    rng = rng_of(11, m)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m), scales(rng, n)
    sa[m // 2], sb[n // 3], sa[0] = np.nan, np.inf, 0
    a[m - 1] = 0
    got = multiply(ctx, a, b, sa, sb, BF16)
    with np.errstate(all="ignore"):
        c = (a.astype(np.int64) @ b.astype(np.int64)) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    assert np.array_equal(np.isnan(c), np.isnan(got)) and np.array_equal(np.isinf(c), np.isinf(got))
    rest = np.delete(np.delete(np.arange(m), [m // 2, m - 1]), []), np.delete(np.arange(n), n // 3)
    at = np.ix_(*rest)
    check_product(got[at], c[at], 3 * 2.0 ** -24 * np.abs(c[at]), BF16)


@pytest.mark.parametrize("m,n,k", [(6, 72, 96), (140, 264, 256), (512, 256, 1024)])
def test_product_with_a_fused_chain(ctx, m, n, k):
    """GELU, then a residual in bf16: every step's result is rounded to its type."""
    rng = rng_of(12, m)
    a, b, sa, sb = codes(rng, m, k), codes(rng, k, n), scales(rng, m) / 20, scales(rng, n)
    bias = HT.from_logical(rng.normal(size=[n]), F32)
    rest = HT.from_logical(rng.normal(size=[m, n]), BF16)
    chain = [(capi.epilogue_op(capi.PW["GELU_FWD"], F32), None),
             (capi.epilogue_op(capi.PW["ADD"], BF16, operand=rest.desc()), rest)]
    got = multiply(ctx, a, b, sa, sb, BF16, bias, epilogue=chain, c_dtype=F32)
    c, bound = product(a, b, sa, sb, bias.logical())
    from math import erf
    gelu = 0.5 * c * (1 + np.vectorize(erf)(c / 2 ** 0.5))
    # (the slope of GELU is at most 1.13; its kernels are good to 2e-6 of the value and 4e-7)
    check_product(got, gelu + rest.logical(), 1.2 * bound + 2e-6 * np.abs(gelu) + 4e-7 + 2 ** -24 * np.abs(rest.logical()), BF16)


# ---- tokens ----------------------------------------------------------------------------
def sample(ctx, logits, uniform, t=None, k=None, p=None, least=None, one=(1.0, 0, 1.0, 0.0), shift=0, fast=None):
    """logits: HT; the settings are vectors or None.  -> (tokens, probabilities)"""
    rows = logits.dims[0]
    d = capi.SampleDesc()
    d.logits = logits.desc()
    d.temperature, d.top_k, d.top_p, d.min_p = one
    vec = {}
    for name, value, dt in (("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32), ("min_p", least, np.float32)):
        setattr(d, "has_" + name, int(value is not None))
        vec[name] = None if value is None else ctx.to_device(np.asarray(value, dt))
    supported = ctx.lib.fhip_sample_supported(d)
    assert supported == (2 if fast else supported if fast is None else 1)
    x = guarded(ctx, logits.storage, shift)
    tok, prob = guarded(ctx, np.full(rows, -77, np.int32)), guarded(ctx, np.full(rows, -7, np.float32))
    room = guarded(ctx, np.full(max(ctx.sample_workspace(d), 1), 0x5A, np.uint8), before=192)
    ctx.sample(d, x[1], ctx.to_device(np.asarray(uniform, np.float32)), tok[1], probability=prob[1], workspace=room[1], **vec)
    room[2]()
    return tok[2](), prob[2]()


def check_tokens(ctx, logits, uniform, t, k, p, least, **kw):
    got, chance = sample(ctx, logits, uniform, t, k, p, least, **kw)
    want, expected = tokens(logits.logical(), uniform, t, k, p, least)
    assert np.array_equal(got, want), [(i, got[i], want[i], t[i], k[i], p[i], least[i]) for i in np.flatnonzero(got != want)][:5]
    # (weights' last places: 2^-40 of the largest; the quotient is rounded once)
    assert (np.abs(chance - expected) <= 2.0 ** -23 * expected + 1e-10).all()


def settings(rng, rows, words):
    return (rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], rows), rng.choice([0, 0, 1, 2, 40, max(1, words // 3), words + 9], rows),
            rng.choice([1.0, 0.95, 0.9, 0.5, 0.1], rows), rng.choice([0.0, 0.0, 0.02, 0.3], rows))


@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("rows,words", [(1, 1), (3, 2), (40, 63), (9, 64), (33, 500), (5, 1025), (3, 4099), (4, 32000), (1, 70001),
                                        (2, 131072), (300, 200), (260, 5000), (130, 9000), (127, 4100), (150, 21000),
                                        (2, 1024), (2, 8192), (2, 8193), (3, 20480), (3, 20481), (1, 1000003)])
def test_sample(ctx, dtype, rows, words):
    rng = rng_of(13, rows, words, dtype)
    x = HT.from_logical(rng.normal(size=[rows, words]) * rng.choice([0.3, 1.5, 4.0], [rows, 1]), dtype)
    check_tokens(ctx, x, rng.random(rows).astype(np.float32), *settings(rng, rows, words), fast=True)
    parts = 1 if rows >= 192 or words <= 20480 else min(-(-512 // rows), -(-words // 4096), 32)
    assert ctx.last_kernel() == f"sample parts={parts}"


@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("layout", ["padded", "columns", "every_second", "odd_address", "one_row_for_all"])
def test_sample_strides(ctx, dtype, layout):
    rows, words = 7, 3001
    rng = rng_of(14, dtype)
    values = rng.normal(size=[rows, words]) * 2
    if layout == "one_row_for_all":
        values[:] = values[:1]
    strides = {"padded": [words + 7, 1], "columns": [1, rows + 1], "every_second": [2 * words, 2], "odd_address": None,
               "one_row_for_all": [0, 1]}[layout]
    x = HT.from_logical(values, dtype, strides)
    check_tokens(ctx, x, rng.random(rows).astype(np.float32), *settings(rng, rows, words),
                 shift=capi.DTYPE_SIZE[dtype] if layout == "odd_address" else 0)


@pytest.mark.parametrize("words", [5, 700, 9000, 40000])
def test_sample_equal_logits(ctx, words):
    """All words alike, two values, and halves: ties go to the lowest index."""
    rng = rng_of(15, words)
    values = np.zeros([8, words])
    values[1] = -7.5
    values[2] = rng.integers(0, 2, words)
    values[3] = rng.integers(-3, 4, words) / 2
    values[4, words // 2:] = -20
    values[5] = np.where(rng.random(words) < 0.5, 0.0, -0.0)
    values[6] = 1e30
    x = HT.from_logical(np.repeat(values, 6, 0), F32)
    n = 48
    t, k, p = np.full(n, 1.0), np.tile([0, 3, 0, words // 2, 0, 0], 8), np.tile([1.0, 1.0, 0.5, 1.0, 0.25, 0.0], 8)
    for u in (0.0, 0.5, 0.75, np.float32(1) - np.float32(2.0 ** -24)):
        check_tokens(ctx, x, np.full(n, u, np.float32), t, k, p, np.tile([0.0, 0.0, 0.0, 0.0, 0.9, 0.0], 8))


@pytest.mark.parametrize("words", [4, 300, 5000, 20000, 24000])
def test_sample_masked_rows(ctx, words):
    """NaN and -inf are never drawn; rows of nothing else have no token; infinities outweigh all."""
    rng = rng_of(16, words)
    x = rng.normal(size=[10, words])
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2], x[2, 1::2] = -np.inf, np.nan
    x[3] = -np.inf
    x[3, words - 1] = -3.4e38
    x[4, rng.random(words) < 0.5] = -np.inf
    x[5, 0] = np.nan
    x[6, 1::3] = np.inf
    x[7] = -3.4028235e38
    x[8] = np.where(rng.random(words) < 0.5, 3.4028235e38, -3.4028235e38)
    x = HT.from_logical(x, F32)
    for i in range(4):
        u = rng.random(10).astype(np.float32)
        check_tokens(ctx, x, u, np.full(10, [1.0, 0.0, 0.7, 2.0][i]), np.full(10, [0, 5, 2, 0][i]), np.full(10, [1.0, 0.9, 0.5, 0.99][i]),
                     np.full(10, [0.0, 0.1, 0.0, 1.0][i]))


@pytest.mark.parametrize("rows,words", [(3, 900), (2, 6000), (2, 18000), (2, 40000), (1, 150000)])
def test_sample_many_words_in_question(ctx, rows, words):
    """Logits so close together, or one so far above, that the words in question are hundreds, thousands or all: each way
    of ordering them, lists that LDS does not hold and rows that no list holds."""
    rng = rng_of(20, rows, words)
    values = rng.normal(size=[rows, words])
    for i in range(rows):
        if i % 3 == 0:
            values[i] *= 1e-3
            values[i, words // 3] = [31.0, 8.0, 2.0][i // 3 % 3]
        elif i % 3 == 1:
            values[i] = np.round(values[i] * 4) / 4
        else:
            values[i, :words // 2] *= 0.01
    x = HT.from_logical(values, F32)
    for j in range(3):
        u = rng.random(rows).astype(np.float32)
        k, p = np.full(rows, [words // 2, 0, words // 3][j]), np.full(rows, [1.0, 0.7, 0.8][j])
        check_tokens(ctx, x, u, np.full(rows, [1.0, 1.0, 4.0][j]), k, p, np.full(rows, [0.0, 0.0, 0.01][j]))


@pytest.mark.parametrize("n", [3, 60, 130, 255, 257, 500, 1000, 1500, 2047, 2049, 3900, 4100, 8000, 8200, 9000])
@pytest.mark.parametrize("words", [24000, 18000])
def test_sample_words_in_question(ctx, words, n):
    """Exactly n words near each other below one that is far above, and nothing else to draw."""
    rng = rng_of(21, words, n)
    values = np.full([2, words], -np.inf)
    for row in values:
        at = rng.choice(words, n + 1, replace=False)
        row[at] = rng.permutation(n + 1) * (1e-3 / n)
        row[at[0]] = 12.0
    x = HT.from_logical(values, F32)
    for u in (0.1, 0.37, 0.99):
        check_tokens(ctx, x, np.full(2, u, np.float32), np.full(2, 1.5), np.array([0, n // 2]), np.array([0.9, 1.0]), np.zeros(2))


def test_calls_are_refused(ctx):
    """What a descriptor does not show: missing pointers, settings without their vector, small or unaligned workspace."""
    d = capi.SampleDesc()
    d.logits, d.temperature, d.top_p = capi.TensorDesc.make([2, 30000], [30000, 1], F32), 1.0, 1.0
    x, u = ctx.to_device(np.zeros([2, 30000], np.float32)), ctx.to_device(np.zeros(2, np.float32))
    _, tok, tokens_back = guarded(ctx, np.full(2, -9, np.int32))
    need = ctx.sample_workspace(d)
    room = ctx.alloc(need + 512)
    at = room.ptr + -room.ptr % 256

    def call(logits=x.ptr, uniform=u.ptr, t=None, token=tok, work=at, size=need):
        return ctx.lib.fhip_sample(ctx.handle, ctypes.byref(d), logits, uniform, t, None, None, None, token, None, work, size)
    for bad in (dict(logits=None), dict(uniform=None), dict(token=None), dict(t=u.ptr), dict(work=None), dict(work=at + 64), dict(size=need - 1)):
        assert call(**bad) != 0, bad
        said = ctx.lib.fhip_last_error(ctx.handle).decode()
        assert "fhip_sample" in said and ("workspace" in said) == bool({"work", "size"} & set(bad)), said
    d.has_top_k = 1
    assert call() != 0
    d.has_top_k = 0
    ctx.sync()
    assert (tokens_back() == -9).all()
    assert call() == 0
    assert (tokens_back() == 0).all()

    q = capi.QuantizeRowsDesc()
    q.x, q.q, q.scale_stride = capi.TensorDesc.make([2, 64], [64, 1], F32), capi.TensorDesc.make([2, 64], [64, 1], capi.INT8), 1
    _, codes, codes_back = guarded(ctx, np.full([2, 64], 5, np.int8))
    run = lambda x, q_, s, up=None, w=None: ctx.lib.fhip_quantize_rows(  # noqa: E731
        ctx.handle, ctypes.byref(q), x, up, w, q_, s, None, 0)
    for bad in ((None, codes, u.ptr), (x.ptr, None, u.ptr), (x.ptr, codes, None), (x.ptr, codes, u.ptr, x.ptr), (x.ptr, codes, u.ptr, None, x.ptr)):
        assert run(*bad) != 0 and "fhip_quantize_rows" in ctx.lib.fhip_last_error(ctx.handle).decode()
    ctx.sync()
    assert (codes_back() == 5).all()
    assert run(x.ptr, codes, u.ptr) == 0 and (codes_back() == 0).all()


def test_sample_many_rows(ctx):
    """More rows than a grid has workgroups of a row each."""
    rows = 2 ** 21 + 5
    x = HT.from_logical(np.tile(np.float32([[0.0, 1.0]]), [rows, 1]), F32)
    got, chance = sample(ctx, x, np.tile(np.float32([0.7, 0.8]), rows // 2 + 1)[:rows])
    assert ctx.last_kernel() == "sample_rows"
    # (1 weighs 1 and comes first, 0 weighs 1 / e: the first up to 0.731)
    assert (got[::2] == 1).all() and (got[1::2] == 0).all()
    assert np.allclose(chance[::2], 1 / (1 + np.exp(-1.0)), rtol=2e-7)


def test_quantize_many_rows(ctx):
    rows = 2 ** 21 + 3
    q, s = quantize(ctx, HT.from_logical(np.tile(np.float32([[3.0], [-5.0], [0.0]]), [rows // 3 + 1, 1])[:rows], F32))
    assert (q[0::3] == 127).all() and (q[1::3] == -127).all() and (q[2::3] == 0).all()
    assert (s[0::3] == np.float32(3) / np.float32(127)).all() and (s[2::3] == 0).all()


# ---- streams, graphs, calls side by side -------------------------------------------------
def serving_step(c, dev, seed, rows=24, k=1024, hidden=2048, words=32768):
    """Norm, codes, product; gate, codes, product onto words; tokens.  -> (run on a context, check)"""
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)
    x = randn(rows, k).to(torch.bfloat16)
    w1 = torch.randint(-127, 128, (2 * hidden, k), generator=gen, device=dev, dtype=torch.int8)
    w2 = torch.randint(-127, 128, (words, hidden), generator=gen, device=dev, dtype=torch.int8)
    s1, s2 = torch.full((2 * hidden,), 4e-4, device=dev), torch.full((words,), 2e-3, device=dev)
    u = torch.rand(rows, generator=gen, device=dev)
    q1, q2 = (torch.empty(rows, n, dtype=torch.int8, device=dev) for n in (k, hidden))
    a1, a2 = (torch.empty(rows, device=dev) for _ in range(2))
    mid, logits = torch.empty(rows, 2 * hidden, dtype=torch.bfloat16, device=dev), torch.empty(rows, words, device=dev)
    token, chance = torch.empty(rows, dtype=torch.int32, device=dev), torch.empty(rows, device=dev)
    T = capi.TensorDesc.make
    n1, n2 = capi.QuantizeRowsDesc(), capi.QuantizeRowsDesc()
    n1.x, n1.q, n1.scale_stride, n1.front, n1.epsilon = T([rows, k], [k, 1], BF16), T([rows, k], [k, 1], capi.INT8), 1, \
        capi.QUANTIZE_FRONT["RMSNORM"], 1e-5
    n2.x, n2.q, n2.scale_stride, n2.front = T([rows, hidden], [2 * hidden, 1], BF16), T([rows, hidden], [hidden, 1], capi.INT8), 1, \
        capi.QUANTIZE_FRONT["SWISH_GATE"]
    n2.up = T([rows, hidden], [2 * hidden, 1], BF16)
    m1, m2 = capi.MatmulQuantizedDesc(), capi.MatmulQuantizedDesc()
    for m, kk, nn, t in ((m1, k, 2 * hidden, BF16), (m2, hidden, words, F32)):
        m.a, m.b, m.c = T([rows, kk], [kk, 1], capi.INT8), T([kk, nn], [1, kk], capi.INT8), T([rows, nn], [nn, 1], t)
        m.out, m.out_dtype, m.a_scale_stride, m.b_scale_stride = m.c, t, 1, 1
    d = capi.SampleDesc()
    d.logits, d.temperature, d.top_k, d.top_p = T([rows, words], [words, 1], F32), 0.9, 50, 0.95
    work = torch.empty(c.sample_workspace(d), dtype=torch.uint8, device=dev)

    def run():
        c.quantize_rows(n1, x.data_ptr(), q1.data_ptr(), a1.data_ptr())
        c.matmul_quantized(m1, q1.data_ptr(), w1.data_ptr(), a1.data_ptr(), s1.data_ptr(), mid.data_ptr())
        c.quantize_rows(n2, mid.data_ptr(), q2.data_ptr(), a2.data_ptr(), up=mid.data_ptr() + 2 * hidden)
        c.matmul_quantized(m2, q2.data_ptr(), w2.data_ptr(), a2.data_ptr(), s2.data_ptr(), logits.data_ptr())
        c.sample(d, logits.data_ptr(), u.data_ptr(), token.data_ptr(), probability=chance.data_ptr(), workspace=work.data_ptr())

    def check():
        codes, scale = q1.cpu().numpy(), a1.cpu().numpy()
        check_codes(codes, scale, *front(x.float().cpu().numpy(), "RMSNORM", eps=1e-5))
        middle = mid.float().cpu().numpy()
        check_product(middle, *product(codes, w1.cpu().numpy().T, scale, s1.cpu().numpy()), BF16)
        y, rel = front(middle[:, :hidden], "SWISH_GATE", up=middle[:, hidden:])
        check_codes(q2.cpu().numpy(), a2.cpu().numpy(), y, rel)
        l = logits.cpu().numpy()
        check_product(l, *product(q2.cpu().numpy(), w2.cpu().numpy().T, a2.cpu().numpy(), s2.cpu().numpy()), F32)
        want, expected = tokens(l, u.cpu().numpy(), [0.9] * rows, [50] * rows, [0.95] * rows, [0.0] * rows)
        assert np.array_equal(token.cpu().numpy(), want)
        assert np.allclose(chance.cpu().numpy(), expected, rtol=2e-7, atol=1e-10)

    def change(seed):
        gen.manual_seed(seed)
        x.copy_(randn(rows, k))
        u.copy_(torch.rand(rows, generator=gen, device=dev))
    return run, check, change


def test_step_on_a_stream_and_captured(ctx):
    """The operators one after another as a decoder uses them: on a stream of the caller's, then captured and replayed with
    other inputs, with other work between the replays."""
    dev = torch.device("cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = capi.Context(torch.cuda.current_device(), stream.cuda_stream)
        run, check, change = serving_step(c, dev, 31)
        stream.synchronize()
        run()
        stream.synchronize()
        check()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
        for i in range(4):
            change(40 + i)
            graph.replay()
            stream.synchronize()
            check()
            run()  # eager work between, of the same operators
            torch.randn(512, 512, device=dev).sum()
            stream.synchronize()
            check()


def test_two_steps_at_once(ctx):
    """Two contexts on streams of their own, with workspaces of their own, side by side."""
    dev = torch.device("cuda")
    steps = []
    for i in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            c = capi.Context(torch.cuda.current_device(), stream.cuda_stream)
            steps.append((c, stream, *serving_step(c, dev, 50 + i, rows=5 + 40 * i)))
    torch.cuda.synchronize()
    for _ in range(6):
        for _, _, run, _, _ in steps:
            run()
    torch.cuda.synchronize()
    for _, _, _, check, _ in steps:
        check()


def test_sample_settings_at_their_ends(ctx):
    rng = rng_of(17)
    words = 3000
    inf, nan = np.inf, np.nan
    rows = [(1.0, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (inf, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0), (1e30, 7, 0.9, 0.0),
            (1.0, -5, 1.0, 0.0), (1.0, 2 ** 31 - 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, nan, 0.0),
            (1.0, 0, inf, 0.0), (1.0, 0, 1.0, nan), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 5.0), (1.0, 0, 1.0, -1.0), (1.0, 0, 1e-30, 0.0),
            (1.0, 0, 0.99999994, 1e-30), (0.01, 1, 0.5, 0.5)]
    t, k, p, least = (np.array(c) for c in zip(*rows))
    x = HT.from_logical(rng.normal(size=[len(rows), words]) * 3, F32)
    for u in (0.0, 0.3, 0.9, np.float32(1) - np.float32(2.0 ** -24)):
        check_tokens(ctx, x, np.full(len(rows), u, np.float32), t, k, p, least)
    # numbers outside [0, 1) count as the nearest inside
    a, _ = sample(ctx, x, np.full(len(rows), 1.5), t, k, p, least)
    b, _ = sample(ctx, x, np.full(len(rows), np.nan), t, k, p, least)
    c, _ = sample(ctx, x, np.full(len(rows), -1.0), t, k, p, least)
    d, _ = sample(ctx, x, np.full(len(rows), 0.0), t, k, p, least)
    assert np.array_equal(b, d) and np.array_equal(c, d)
    assert a[2] == d[2] and a[0] != d[0]


def test_sample_settings_of_the_descriptor(ctx):
    rng = rng_of(18)
    x = HT.from_logical(rng.normal(size=[20, 900]) * 2, BF16)
    u = rng.random(20).astype(np.float32)
    got, chance = sample(ctx, x, u, one=(0.8, 30, 0.9, 0.01))
    want, expected = tokens(x.logical(), u, [0.8] * 20, [30] * 20, [0.9] * 20, [0.01] * 20)
    assert np.array_equal(got, want) and np.allclose(chance, expected, rtol=2e-7, atol=0)


def test_sample_covers_the_distribution(ctx):
    """4096 evenly spaced numbers draw every word as often as its probability says, off by one at most."""
    rng = rng_of(19)
    n, words = 4096, 50
    logits = rng.normal(size=words).astype(np.float32)
    x = HT.from_logical(np.broadcast_to(logits, [n, words]), F32, [0, 1])
    got, chance = sample(ctx, x, (np.arange(n) + 0.5) / n)
    w = np.exp(logits.astype(np.float64) - logits.max())
    w /= w.sum()
    assert (np.abs(np.bincount(got, minlength=words) - n * w) <= 1.01).all()
    assert np.allclose(chance, w[got], rtol=3e-7)


# ---- the C++ graph API -------------------------------------------------------------------
def test_graphs():
    cpp_binary("test_quantized_api", 120)
