"""What the packed and paged operators refuse, and what they say; no GPU."""
import ctypes

import numpy as np
import pytest

from fusilli_amd import capi
from serving import cpp_binary, from_groups, to_groups

LIB = capi.load()


def rows(t, h, d, dtype=capi.BFLOAT16, strides=None):
    return capi.TensorDesc.make([t, h, d], strides or [h * d, d, 1], dtype)


def pool(p, h, s, d, dtype=capi.BFLOAT16, strides=None):
    return capi.TensorDesc.make([p, h, s, d], strides or [h * s * d, s * d, d, 1], dtype)


def cache(d=128, heads=2, page=16, dtype=capi.BFLOAT16, group=0, dv=None, batch=3):
    c = capi.CacheDesc()
    dv = dv or d
    if group:
        c.k, c.v = pool(9, heads, page, d // 2, capi.UINT8), pool(9, heads, page, dv // 2, capi.UINT8)
        c.k_params, c.v_params = (pool(9, heads, page, 2 * x // group, capi.HALF) for x in (d, dv))
    else:
        c.k, c.v = pool(9, heads, page, d, dtype), pool(9, heads, page, dv, dtype)
    c.batch, c.pages_per_sequence, c.page_stride = batch, 4, 4
    return c


def packed(d=128, dtype=capi.BFLOAT16):
    x = capi.SdpaPackedDesc()
    x.q, x.k, x.v, x.o = rows(50, 8, d, dtype), rows(50, 2, d, dtype), rows(50, 2, d, dtype), rows(50, 8, d, dtype)
    x.batch, x.is_causal = 3, 1
    return x


def paged(d=128, dtype=capi.BFLOAT16, group=0, page=16):
    x = capi.SdpaPagedDesc()
    x.q, x.o, x.cache, x.is_causal = rows(3, 8, d, dtype), rows(3, 8, d, dtype), cache(d, page=page, dtype=dtype, group=group), 1
    return x


def append(d=128, dtype=capi.BFLOAT16, group=0):
    x = capi.CacheAppendDesc()
    x.k, x.v, x.k_out = rows(50, 2, d, dtype), rows(50, 2, d, dtype), rows(50, 2, d, dtype)
    x.q, x.q_out = rows(50, 8, d, dtype), rows(50, 8, d, dtype)
    x.rotation = capi.TensorDesc.make([100, d], [d, 1], capi.FLOAT)
    x.cache = cache(d, dtype=dtype, group=group)
    return x


def read(d=128, dtype=capi.BFLOAT16, group=0):
    x = capi.CacheReadDesc()
    x.k, x.v, x.cache = rows(50, 2, d, dtype), rows(50, 2, d, dtype), cache(d, dtype=dtype, group=group)
    return x


SUPPORTED = {"packed": LIB.fhip_sdpa_packed_fwd_supported, "paged": LIB.fhip_sdpa_paged_fwd_supported,
             "append": LIB.fhip_cache_append_supported, "read": LIB.fhip_cache_read_supported}
MAKE = {"packed": packed, "paged": paged, "append": append, "read": read}


def put(x, path, value):
    *to, last = path.split(".")
    for name in to:
        x = getattr(x, name)
    setattr(x, last, value)


REFUSED = [
    ("packed", "q", rows(50, 7, 128), "no multiple"),
    ("packed", "k", rows(51, 2, 128), "differ in rows"),
    ("packed", "k", rows(50, 2, 128, capi.HALF), "differ in type"),
    ("packed", "k", rows(50, 2, 64), "head dim"),
    ("packed", "v", rows(50, 2, 64), "O must be"),
    ("packed", "o", rows(50, 8, 128, capi.FLOAT), "O must be"),
    ("packed", "o", rows(50, 8, 128, strides=[0, 128, 1]), "stride of 0"),
    ("packed", "q", rows(50, 8, 128, strides=[2048, 256, 2]), "unit stride"),
    ("packed", "q", rows(50, 8, 128, capi.DOUBLE), "f32, bf16 or f16"),
    ("packed", "q", pool(1, 50, 8, 128), "rank 3"),
    ("packed", "batch", 0, "batch"),
    ("packed", "v", rows(50, 2, 1024), "out of range"),
    ("paged", "q", rows(3, 7, 128), "no multiple"),
    ("paged", "o", rows(3, 8, 64), "head dims"),
    ("paged", "cache.k", pool(9, 2, 16, 64), "head dims"),
    ("paged", "cache.v", pool(9, 2, 32, 128), "differ in dim 2"),
    ("paged", "cache.v", pool(9, 2, 16, 128, capi.HALF), "differ in type"),
    ("paged", "cache", cache(dtype=capi.HALF), "rows' type"),
    ("paged", "cache.k_params", pool(9, 2, 16, 4, capi.HALF), "parameters go"),
    ("paged", "cache.batch", 0, "batch"),
    ("paged", "cache.pages_per_sequence", 1 << 40, "2^30 keys"),
    ("paged", "cache.pages_per_sequence", 0, "2^30 keys"),
    ("paged", "cache.page_stride", 3, "overlap"),
    ("append", "v", rows(49, 2, 128), "differ in rows"),
    ("append", "q", rows(50, 8, 64), "Q_OUT dims"),
    ("append", "q_out", capi.TensorDesc.absent(), "go together"),
    ("append", "k_out", rows(50, 2, 128, capi.HALF), "another type"),
    ("append", "k_out", rows(50, 2, 128, strides=[256, 0, 1]), "stride of 0"),
    ("append", "rotation", capi.TensorDesc.make([100, 130], [130, 1], capi.FLOAT), "130 of 128"),
    ("append", "rotation", capi.TensorDesc.make([100, 63], [63, 1], capi.FLOAT), "63 of 128"),
    ("append", "rotation", capi.TensorDesc.make([100, 64], [64, 1], capi.HALF), "must be Float"),
    ("append", "cache", cache(heads=4), "4 heads"),
    ("append", "cache.k", pool(9, 2, 16, 128, strides=[0, 2048, 128, 1]), "stride of 0"),
    ("read", "v", rows(50, 4, 128), "differ in rows"),
    ("read", "cache.k", pool(9, 2, 16, 128, strides=[8192, 4096, 256, 2]), "unit stride"),
    ("read", "cache.k", capi.TensorDesc.make([9, 2, 128], [256, 128, 1], capi.BFLOAT16), "rank 4"),
]


@pytest.mark.parametrize("what,field,value,says", REFUSED)
def test_refused(what, field, value, says):
    x = MAKE[what]()
    assert SUPPORTED[what](x) > 0
    put(x, field, value)
    assert SUPPORTED[what](x) == 0
    assert says in LIB.fhip_last_error(None).decode()


@pytest.mark.parametrize("what", ["paged", "append", "read"])
@pytest.mark.parametrize("field,value,says", [
    ("cache.k_params", pool(9, 2, 16, 5, capi.HALF), "groups must"),
    ("cache.k_params", pool(9, 2, 16, 6, capi.HALF), "groups must"),
    ("cache.k_params", pool(9, 2, 16, 8, capi.HALF), "groups must"),      # not V's
    ("cache.k_params", pool(9, 2, 16, 4, capi.BFLOAT16), "must be Half"),
    ("cache.v_params", pool(9, 2, 8, 4, capi.HALF), "must be Half"),
    ("cache.v_params", capi.TensorDesc.absent(), "parameters go"),
    ("cache.v", pool(9, 2, 16, 128, capi.UINT8), "head dims"),
])
def test_refused_in_4_bits(what, field, value, says):
    x = MAKE[what](group=64)
    assert SUPPORTED[what](x) > 0
    put(x, field, value)
    assert SUPPORTED[what](x) == 0
    assert says in LIB.fhip_last_error(None).decode()


@pytest.mark.parametrize("what", sorted(MAKE))
@pytest.mark.parametrize("d,dtype", [(128, capi.BFLOAT16), (64, capi.HALF), (80, capi.BFLOAT16), (128, capi.FLOAT), (512, capi.HALF)])
def test_taken(what, d, dtype):
    assert SUPPORTED[what](MAKE[what](d, dtype)) > 0
    assert SUPPORTED[what](None) == 0


@pytest.mark.parametrize("what", ["packed", "paged"])
@pytest.mark.parametrize("scale,level", [(1e8, 2), (1e-30, 2), (1.1e8, 1), (3e38, 1), (np.inf, 1), (np.nan, 1), (0.0, 1), (-1.0, 1)])
def test_scales_of_the_tuned_kernels(what, scale, level):
    x = MAKE[what]()
    x.has_scale, x.scale = 1, scale
    assert SUPPORTED[what](x) == level
    x.has_scale = 0  # (then it is not read)
    assert SUPPORTED[what](x) == 2


def test_null_arguments():
    n = ctypes.c_size_t(1)
    for name, make in (("sdpa_packed_fwd", packed), ("sdpa_paged_fwd", paged), ("cache_append", append), ("cache_read", read)):
        size = getattr(LIB, f"fhip_{name}_workspace_size")
        assert size(None, ctypes.byref(n)) != 0 and size(make(), None) != 0
        assert size(make(), ctypes.byref(n)) == 0
    assert LIB.fhip_sdpa_packed_fwd(None, packed(), *[None] * 7, 0) != 0
    assert LIB.fhip_sdpa_paged_fwd(None, paged(), None, *[None] * 4, 0) != 0
    assert LIB.fhip_cache_append(None, append(), None, *[None] * 9, 0) != 0
    assert LIB.fhip_cache_read(None, read(), None, *[None] * 4, 0) != 0
    assert "null context" in LIB.fhip_last_error(None).decode()


def test_descriptors_have_the_c_layout():
    t = ctypes.sizeof(capi.TensorDesc)
    assert ctypes.sizeof(capi.CacheDesc) == 4 * t + 24
    assert ctypes.sizeof(capi.CachePointers) == 48
    assert ctypes.sizeof(capi.SdpaPackedDesc) == 4 * t + 24
    assert ctypes.sizeof(capi.SdpaPagedDesc) == 6 * t + 24 + 16
    assert ctypes.sizeof(capi.CacheAppendDesc) == 10 * t + 24 + 8
    assert ctypes.sizeof(capi.CacheReadDesc) == 6 * t + 24


def test_the_formula_of_4_bits_keeps_within_half_a_scale():
    # |x - value| <= scale / 2, and what low and scale lost to half: low's half step, 15 half steps of the scale
    x = np.random.default_rng(0).standard_normal([40, 128]).astype(np.float32)
    code, scale, low = to_groups(x, 32)
    far = np.repeat(scale.astype(np.float64) * (0.5 + 15 * 2.0 ** -11) + np.abs(low.astype(np.float64)) * 2.0 ** -11, 32, -1)
    assert (np.abs(from_groups(code, scale, low) - x) <= far * (1 + 1e-5)).all()
    assert code.max() == 15 and code.min() == 0


# -- the C++ graph API (tests/cpp/test_serving_api.cpp) -------------------------
def test_graph_api_on_the_host():
    cpp_binary("test_serving_api", 120, "host")


def test_rows_of_any_offsets_on_the_host():
    cpp_binary("test_serving_split", 60)
