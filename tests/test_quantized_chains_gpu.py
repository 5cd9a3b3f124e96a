"""Scaled products of codes with chains over columns and results of every type, on each family of kernels."""
import numpy as np
import pytest
import torch  # noqa: F401 (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
from quantized import HALF_STEP, UNIT, check_product, guarded

pytestmark = pytest.mark.gpu
BF16, F16, F32 = capi.BFLOAT16, capi.HALF, capi.FLOAT
NAME = {BF16: "bf16", F16: "f16", F32: "f32"}


@pytest.mark.parametrize("m,n,k", [(5, 72, 96), (130, 257, 40), (140, 264, 256), (256, 384, 512), (512, 512, 4096), (1024, 1280, 2048)])
@pytest.mark.parametrize("c_dtype,dtype", [(F32, BF16), (BF16, F32), (F16, BF16), (BF16, BF16), (F32, F32), (F32, F16)],
                         ids=lambda d: NAME[d])
def test_columns_multiplied_cut_and_added(ctx, m, n, k, c_dtype, dtype):
    """relu(C w) + t with w and t along the columns, each step in f32, the last rounded to OUT's type."""
    rng = np.random.default_rng([m, n, k, c_dtype, dtype])
    a, b = (rng.integers(-128, 128, s, np.int8) for s in ([m, k], [k, n]))
    sa, sb = ((0.5 + rng.random(s)).astype(np.float32) * np.float32(0.01) for s in (m, n))
    sb *= np.float32(k ** -0.5)
    w, t = HT.from_logical(1 + rng.random([1, n]), F32), HT.from_logical(rng.normal(size=[1, n]), BF16)
    hb, out = HT.from_logical(b, capi.INT8, [1, k]), HT.empty([m, n], dtype, [n + 8, 1], fill=3)
    d = capi.MatmulQuantizedDesc()
    d.a, d.b, d.c = capi.TensorDesc.make([m, k], [k, 1], capi.INT8), hb.desc(), capi.TensorDesc.make([m, n], [n, 1], c_dtype)
    d.out, d.out_dtype, d.a_scale_stride, d.b_scale_stride = out.desc(), dtype, 1, 1
    d.epilogue = capi.make_epilogue([capi.epilogue_op(capi.PW["MUL"], F32, operand=w.desc(), operand_index=0),
                                     capi.epilogue_op(capi.PW["RELU_FWD"], F32),
                                     capi.epilogue_op(capi.PW["ADD"], dtype, operand=t.desc(), operand_index=1)])
    keep = [ctx.to_device(x) for x in (a, hb.storage, sa, sb, w.storage, t.storage)]
    o = guarded(ctx, out.storage)
    ctx.matmul_quantized(d, *keep[:4], o[1], epilogue_operands=keep[4:])
    out.storage = o[2]()
    # (whole sums are exact in f64; the sum in f32, its first product and its second round once each)
    c = a.astype(np.float64) @ b.astype(np.float64) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    bound = 3 * UNIT * np.abs(c) * 1.001
    bound = bound + HALF_STEP[c_dtype] * (np.abs(c) + bound) + (2.0 ** -25 if c_dtype == F16 else 0)
    by = np.asarray(w.logical(), np.float64)
    y = np.maximum(c * by, 0) + t.logical()
    # (the product and the sum round once each, or once together)
    check_product(out.logical(), y, bound * by + UNIT * (np.abs(c * by) * 1.01 + np.abs(y)), dtype)


@pytest.mark.parametrize("m,n,k", [(1000, 1100, 15), (1000, 1100, 16), (1024, 2048, 64), (1500, 1032, 100), (2050, 1300, 127), (1152, 1024, 128)])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=NAME.get)
@pytest.mark.parametrize("along_k", [True, False])
def test_many_results_of_a_short_reduction(ctx, m, n, k, dtype, along_k):
    rng = np.random.default_rng([m, n, k])
    a, b = (rng.integers(-128, 128, s, np.int8) for s in ([m, k], [k, n]))
    sa, sb = ((0.5 + rng.random(s)).astype(np.float32) * np.float32(0.01) for s in (m, n))
    hb, out = HT.from_logical(b, capi.INT8, [1, k] if along_k else None), HT.empty([m, n], dtype, [n + 3, 1], fill=3)
    d = capi.MatmulQuantizedDesc()
    d.a, d.b, d.c = capi.TensorDesc.make([m, k], [k, 1], capi.INT8), hb.desc(), capi.TensorDesc.make([m, n], [n, 1], dtype)
    d.out, d.out_dtype, d.a_scale_stride, d.b_scale_stride = out.desc(), dtype, 1, 1
    o = guarded(ctx, out.storage)
    ctx.matmul_quantized(d, *[ctx.to_device(x) for x in (a, hb.storage, sa, sb)], o[1])
    out.storage = o[2]()
    assert (out.storage[: (m - 1) * (n + 3)].reshape(m - 1, n + 3)[:, n:] == 3).all()
    c = a.astype(np.float64) @ b.astype(np.float64) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    check_product(out.logical(), c, 3 * UNIT * np.abs(c) * 1.001, dtype)
