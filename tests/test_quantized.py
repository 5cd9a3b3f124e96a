"""What the operators of models served in 8 bits refuse, and what they say; no GPU."""
import ctypes

import numpy as np
import pytest

from fusilli_amd import capi
from quantized import codes_in_f32, matrix, token
from serving import cpp_binary

LIB = capi.load()
BF16, F16, F32, I8 = capi.BFLOAT16, capi.HALF, capi.FLOAT, capi.INT8


def quantize(front="NONE"):
    d = capi.QuantizeRowsDesc()
    d.x, d.q, d.scale_stride, d.front = matrix([50, 256], BF16), matrix([50, 256], I8), 1, capi.QUANTIZE_FRONT[front]
    if front == "SWISH_GATE":
        d.up = matrix([50, 256], BF16)
    if front == "RMSNORM":
        d.has_weight, d.weight_dtype, d.weight_stride, d.epsilon = 1, BF16, 1, 1e-6
    return d


def product(dtype=BF16):
    d = capi.MatmulQuantizedDesc()
    d.a, d.b, d.c, d.out = matrix([200, 256], I8), matrix([256, 384], I8, [1, 256]), matrix([200, 384], dtype), matrix([200, 384], dtype)
    d.out_dtype, d.a_scale_stride, d.b_scale_stride = dtype, 1, 1
    return d


def sample(dtype=F32):
    d = capi.SampleDesc()
    d.logits, d.temperature, d.top_p = matrix([4, 1000], dtype), 1.0, 1.0
    return d


SUPPORTED = {"quantize": LIB.fhip_quantize_rows_supported, "gate": LIB.fhip_quantize_rows_supported,
             "rms": LIB.fhip_quantize_rows_supported, "product": LIB.fhip_matmul_quantized_supported,
             "sample": LIB.fhip_sample_supported}
MAKE = {"quantize": quantize, "gate": lambda: quantize("SWISH_GATE"), "rms": lambda: quantize("RMSNORM"),
        "product": product, "sample": sample}

REFUSED = [
    ("quantize", "x", matrix([50, 256], I8), "f32, bf16 or f16"),
    ("quantize", "x", matrix([51, 256], BF16), "[rows, K]"),
    ("quantize", "x", capi.TensorDesc.make([50, 2, 128], [256, 128, 1], BF16), "[rows, K]"),
    ("quantize", "q", matrix([50, 256], capi.UINT8), "Int8"),
    ("quantize", "q", matrix([50, 256], I8, [0, 1]), "stride of 0"),
    ("quantize", "q", matrix([50, 256], I8, [256, 0]), "stride of 0"),
    ("quantize", "scale_stride", 0, "scale_stride"),
    ("quantize", "scale_stride", -1, "scale_stride"),
    ("quantize", "front", 3, "unknown front"),
    ("quantize", "front", -1, "unknown front"),
    ("quantize", "up", matrix([50, 256], BF16), "go together"),
    ("quantize", "has_weight", 1, "needs the RMS norm"),
    ("gate", "up", capi.TensorDesc(), "go together"),
    ("gate", "up", matrix([50, 255], BF16), "X's dims and type"),
    ("gate", "up", matrix([50, 256], F16), "X's dims and type"),
    ("rms", "weight_dtype", I8, "weight must be"),
    ("rms", "weight_stride", -1, "weight must be"),
    ("rms", "epsilon", -1.0, "epsilon"),
    ("rms", "epsilon", float("nan"), "epsilon"),
    ("product", "a", matrix([200, 256], capi.UINT8), "Int8"),
    ("product", "b", matrix([256, 384], BF16), "Int8"),
    ("product", "b", matrix([255, 384], I8), "K mismatch"),
    ("product", "a", capi.TensorDesc.make([1, 200, 256], [51200, 256, 1], I8), "matrices"),
    ("product", "c", matrix([200, 384], capi.INT32), "C must be"),
    ("product", "c", matrix([201, 384], BF16), "M x N"),
    ("product", "out", matrix([200, 383], BF16), "OUT dims"),
    ("product", "out", matrix([200, 384], F32), "out_dtype"),
    ("product", "out", matrix([200, 384], BF16, [384, 0]), "stride of 0"),
    ("product", "a_scale_stride", -1, "between scales"),
    ("product", "b_scale_stride", -1, "between scales"),
    ("sample", "logits", capi.TensorDesc.make([1000], [1], F32), "[rows, words]"),
    ("sample", "logits", matrix([4, 1000], capi.INT32), "f32, bf16 or f16"),
    ("sample", "logits", matrix([4, (1 << 24) + 1], F32), "2^24"),
    ("sample", "logits", matrix([4, 0], F32), "dim[1]=0"),
]


@pytest.mark.parametrize("which,field,value,says", REFUSED, ids=[f"{w}-{f}-{i}" for i, (w, f, _, _) in enumerate(REFUSED)])
def test_refused(which, field, value, says):
    d = MAKE[which]()
    assert SUPPORTED[which](d) > 0
    setattr(d, field, value)
    assert SUPPORTED[which](d) == 0
    assert says in LIB.fhip_last_error(None).decode()


def test_longest_reduction():
    d = product()
    for k, fine in ((131071, True), (131072, False)):
        d.a, d.b = matrix([200, k], I8), matrix([k, 384], I8)
        assert (SUPPORTED["product"](d) > 0) == fine
    assert "131071" in LIB.fhip_last_error(None).decode()


def test_bias_and_chain_are_checked():
    d = product()
    d.has_bias, d.bias_dtype, d.bias_stride = 1, I8, 1
    assert SUPPORTED["product"](d) == 0 and "bias must be" in LIB.fhip_last_error(None).decode()
    d.bias_dtype = F32
    assert SUPPORTED["product"](d) > 0


def test_null_arguments_are_refused():
    n = ctypes.c_size_t(0)
    for name, make in (("quantize_rows", quantize), ("matmul_quantized", product), ("sample", sample)):
        size = getattr(LIB, f"fhip_{name}_workspace_size")
        assert size(None, n) != 0 and size(make(), None) != 0 and size(make(), n) == 0
        assert getattr(LIB, f"fhip_{name}_supported")(None) == 0
    assert LIB.fhip_quantize_rows(None, quantize(), *[None] * 6, 0) != 0
    assert "null context" in LIB.fhip_last_error(None).decode()
    assert LIB.fhip_matmul_quantized(None, product(), *[None] * 8, 0) != 0
    assert LIB.fhip_sample(None, sample(), *[None] * 9, 0) != 0


def test_descriptors_have_the_c_layout():
    t, e = ctypes.sizeof(capi.TensorDesc), ctypes.sizeof(capi.Epilogue)
    assert ctypes.sizeof(capi.QuantizeRowsDesc) == 3 * t + 32
    assert ctypes.sizeof(capi.MatmulQuantizedDesc) == 4 * t + e + 8 + 24 + 8
    assert ctypes.sizeof(capi.SampleDesc) == t + 32


def test_the_formulas_on_known_rows():
    q, s = codes_in_f32(np.array([[127, -127, 1, 0.4, 0.6, 0]]))
    assert q.tolist() == [[127, -127, 1, 0, 1, 0]] and s.tolist() == [1]
    q, s = codes_in_f32(np.array([[0.0, 0], [2.0 ** -130, -2.0 ** -131]]))
    assert q.tolist() == [[0, 0], [127, -64]] and s[0] == 0
    l = np.log([1, 4, 2, 1, 0.5])  # weights 4, 2, 1, 1, 0.5 in order 1, 2, 0, 3, 4
    assert [token(l, u)[0] for u in (0, 0.46, 0.48, 0.69, 0.71, 0.81, 0.83, 0.99)] == [1, 1, 2, 2, 0, 0, 3, 4]
    assert token(l, 0.99, k=2) == (2, pytest.approx(2 / 6))
    assert token(l, 0.99, p=0.8)[0] == 0 and token(l, 0.99, least=0.3)[0] == 2 and token(l, 0.99, t=0) == (1, 1.0)
    assert token([-np.inf, np.nan], 0.5) == (-1, 0.0)


# -- the C++ graph API (tests/cpp/test_quantized_api.cpp) -------------------------
def test_cpp_nodes_and_plans():
    cpp_binary("test_quantized_api", 120, "host")
