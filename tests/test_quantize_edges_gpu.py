"""Rows to codes behind an RMS norm without an epsilon."""
import numpy as np
import pytest
import torch  # noqa: F401 (before the library, which then shares its runtime)

from fusilli_amd import capi
from helpers import HT
from quantized import check_codes, front

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,step", [(96, 1), (1024, 1), (1024, 2), (40000, 1)])
@pytest.mark.parametrize("dtype", [capi.BFLOAT16, capi.FLOAT], ids=["bf16", "f32"])
def test_squares_below_f32(ctx, dtype, k, step):
    """Squares that are all 0 leave nothing to divide by: such a row counts as not finite.  Others are as ever."""
    x = np.random.default_rng(k).normal(size=[4, k])
    x[1] *= 1e-25
    x[2] = 0
    x[3] *= 1e-12
    x = HT.from_logical(x, dtype, [step * k, step])
    d = capi.QuantizeRowsDesc()
    d.x, d.q, d.scale_stride = x.desc(), capi.TensorDesc.make([4, k], [k, 1], capi.INT8), 1
    d.front, d.epsilon = capi.QUANTIZE_FRONT["RMSNORM"], 0.0
    q, s = ctx.to_device(np.full([4, k], 99, np.int8)), ctx.to_device(np.full(4, -5, np.float32))
    ctx.quantize_rows(d, x.upload(ctx), q, s)
    assert ctx.last_kernel() == ("quantize_rows_held" if step == 1 and k <= 32768 else "quantize_rows_generic")
    codes, scales = q.download(np.int8).reshape(4, k), s.download(np.float32)
    assert np.isnan(scales[[1, 2]]).all() and not codes[[1, 2]].any()
    y, rel = front(x.logical()[[0, 3]], "RMSNORM", eps=0.0)
    check_codes(codes[[0, 3]], scales[[0, 3]], y, rel)
