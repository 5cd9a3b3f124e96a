// A key / value cache in pages: appending packed rows to it, positions rotated
// into queries and keys on the way, and reading rows back.
//
// Bound by the bytes of the rows, read once and written once.  Kernels for 16-bit
// rows on 16 bytes: a lane owns 8 elements, the lanes of a row lie side by side, a
// wavefront takes the same few heads of neighbouring rows, so that a row's
// angles are loaded once for them; sequences are found with one load of offsets in all lanes and a
// ballot per row, beside the rows' own loads, and only the page and the angles wait for that.  A group in
// 4 bits is a few neighbouring lanes, whose minimum and maximum meet by DPP.  bf16, 32 query and 8 key heads of
// 128: 18997 rows into 16 bits 103.5 us, 5.0 TB/s; 15036 into 4 bits 83.6 us, 4.4 TB/s; 26656 out of 4 bits 33.7 us,
// 4.2 TB/s.  Seven tokens 5.1 us, which is one launch.
//
// Kernels for any type, size and stride: one wavefront per row of one head.  18997 rows of 36 dims 0.59 ms, 0.25 TB/s.
#include "paged_cache.h"
#include "fast_paths.h"

#include <cmath>
#include <type_traits>

namespace {

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out, *k_out;
  const float *rotation;
  const int32_t *offsets, *positions;
  FhipCacheView cache;
  int64_t q_s[2], k_s[2], v_s[2], qo_s[2], ko_s[2]; // row and head strides
  int64_t rot_s;
  int32_t dtype, T, Hq, Hkv, D, Dv, R, table_rows, interleaved;
};

// Rounds a group's values (in LDS) and stores a row of a pool.
__device__ void store_row(const FhipCacheView &c, const FhipPool &p, int page, int slot, int h, const float *x, int D,
                          int lane) {
  const int64_t at = page * p.page + h * p.head + slot * p.slot;
  if (!c.group) {
    for (int e = lane; e < D; e += 64)
      fhip_store<float>(p.data, c.dtype, at + e, x[e]);
    return;
  }
  _Float16 *pairs = p.params + page * p.params_page + h * p.params_head + slot * p.params_slot;
  for (int e = lane * 2; e < D; e += 128) {
    const float *of = x + e / c.group * c.group;
    float lo = of[0], hi = of[0];
    bool number = true;
    for (int i = 0; i < c.group; ++i) {
      lo = fminf(lo, of[i]), hi = fmaxf(hi, of[i]);
      number &= __builtin_fabsf(of[i]) < INFINITY;
    }
    const FhipGroup g = fhip_group_of(number ? lo : INFINITY, hi);
    ((uint8_t *)p.data)[at + e / 2] = (uint8_t)((uint32_t)fhip_code_of(g, x[e]) | (uint32_t)fhip_code_of(g, x[e + 1]) << 4);
    if (e % c.group == 0)
      pairs[e / c.group * 2] = g.scale, pairs[e / c.group * 2 + 1] = g.low;
  }
}

__global__ __launch_bounds__(64) void append_rows_kernel(AppendArgs g) {
#pragma clang fp contract(off)
  __shared__ float row[kCacheMaxDim];
  const int heads = g.Hq + 2 * g.Hkv;
  const uint32_t at_line = fhip_line_index(blockIdx.y);
  const int t = (int)(at_line / (uint32_t)heads), which = (int)(at_line % (uint32_t)heads);
  const int lane = threadIdx.x;
  if (t >= g.T)
    return;
  const int b = fhip_sequence_of(g.offsets, g.cache.batch, t);
  if (b < 0)
    return;
  const int64_t place = (int64_t)g.cache.lengths[b] - g.offsets[b + 1] + t;
  const int64_t pos = g.positions ? g.positions[t] : place;
  const bool turned = !g.R || (pos >= 0 && pos < g.table_rows);
  const int page = place >= 0 && place < kCacheMaxKeys ? fhip_page_of(g.cache, b, (int)place) : -1;
  const int slot = page < 0 ? 0 : (int)(place % g.cache.page_size);
  if (which >= g.Hq + g.Hkv) { // a row of V
    const int h = which - g.Hq - g.Hkv;
    if (page < 0 || !turned)
      return;
    for (int e = lane; e < g.Dv; e += 64)
      row[e] = fhip_load<float>(g.v, g.dtype, t * g.v_s[0] + h * g.v_s[1] + e);
    __syncthreads();
    store_row(g.cache, g.cache.v, page, slot, h, row, g.Dv, lane);
    return;
  }
  const bool is_q = which < g.Hq;
  const int h = is_q ? which : which - g.Hq;
  const void *x = is_q ? g.q : g.k;
  const int64_t at = t * (is_q ? g.q_s[0] : g.k_s[0]) + h * (is_q ? g.q_s[1] : g.k_s[1]);
  const float *angles = g.R && turned ? g.rotation + pos * g.rot_s : nullptr;
  const int half = g.R / 2;
  for (int e = lane; e < g.D; e += 64) {
    float y = fhip_load<float>(x, g.dtype, at + e);
    if (e < g.R) {
      // (the pair's first and second element, each with its own sign)
      const int i = g.interleaved ? e >> 1 : e % half;
      const bool second = g.interleaved ? e & 1 : e >= half;
      const int other = g.interleaved ? e ^ 1 : second ? e - half : e + half;
      const float z = fhip_load<float>(x, g.dtype, at + other);
      if (angles) {
        const float c = angles[i], s = angles[half + i];
        const float yc = y * c, zs = z * s;
        y = second ? yc + zs : yc - zs;
      }
    }
    row[e] = turned ? fhip_round_through<float>(g.dtype, y) : __builtin_nanf("");
  }
  __syncthreads();
  void *out = is_q ? g.q_out : g.k_out;
  if (out) {
    const int64_t to = t * (is_q ? g.qo_s[0] : g.ko_s[0]) + h * (is_q ? g.qo_s[1] : g.ko_s[1]);
    for (int e = lane; e < g.D; e += 64)
      fhip_store<float>(out, g.dtype, to + e, row[e]);
  }
  if (!is_q && page >= 0 && turned)
    store_row(g.cache, g.cache.k, page, slot, h, row, g.D, lane);
}

struct ReadArgs {
  void *k, *v;
  const int32_t *offsets;
  FhipCacheView cache;
  int64_t k_s[2], v_s[2];
  int32_t dtype, T, Hkv, D, Dv;
};

__global__ __launch_bounds__(64) void read_rows_kernel(ReadArgs g) {
  const uint32_t at_line = fhip_line_index(blockIdx.y);
  const int t = (int)(at_line / (uint32_t)(2 * g.Hkv)), which = (int)(at_line % (uint32_t)(2 * g.Hkv));
  if (t >= g.T)
    return;
  const int b = fhip_sequence_of(g.offsets, g.cache.batch, t);
  if (b < 0)
    return;
  const int64_t place = (int64_t)g.cache.lengths[b] - g.offsets[b + 1] + t;
  const int page = place >= 0 && place < kCacheMaxKeys ? fhip_page_of(g.cache, b, (int)place) : -1;
  const int slot = page < 0 ? 0 : (int)(place % g.cache.page_size);
  const bool is_k = which < g.Hkv;
  const int h = is_k ? which : which - g.Hkv, D = is_k ? g.D : g.Dv;
  const FhipPool &p = is_k ? g.cache.k : g.cache.v;
  void *out = is_k ? g.k : g.v;
  const int64_t to = t * (is_k ? g.k_s[0] : g.v_s[0]) + h * (is_k ? g.k_s[1] : g.v_s[1]);
  for (int e = threadIdx.x; e < D; e += 64)
    fhip_store<float>(out, g.dtype, to + e,
                      page < 0 ? __builtin_nanf("") : fhip_cache_value(g.cache, p, page, slot, h, e));
}

// ---- 16-bit rows, 8 elements per lane ---------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kThreads = 256;

template <bool BF16> __device__ __forceinline__ void widen(const u32x4 &x, float (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = x[i / 2]; // (through a scalar: bit-casting a vector's element in place reads element 0)
    if constexpr (BF16)
      y[i] = __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
    else
      y[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w));
  }
}
template <bool BF16> __device__ __forceinline__ u32x4 narrow(const float (&y)[8]) {
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      x[i] = __builtin_bit_cast(uint32_t, b2{(__bf16)y[2 * i], (__bf16)y[2 * i + 1]});
    } else {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      x[i] = __builtin_bit_cast(uint32_t, h2{(_Float16)y[2 * i], (_Float16)y[2 * i + 1]});
    }
  }
  return x;
}

// A lane's row: its sequence (-1: none) and place.  All lanes call it; `t` is the same in the lanes of a row.
struct RowPlace {
  int b;
  int64_t place;
};
template <int LANES>
__device__ __forceinline__ RowPlace place_of(const FhipCacheView &c, const int32_t *offsets, int t, bool in) {
  const int l = threadIdx.x & 63;
  if (c.batch <= 64) {
    const int end = l < c.batch ? offsets[l + 1] : INT32_MAX, length = l < c.batch ? c.lengths[l] : 0;
    const int start = offsets[0];
    int b = 0;
#pragma unroll
    for (int r = 0; r < 64 / LANES; ++r) { // sequences that end in front of row r of this wavefront
      const int row = __builtin_amdgcn_readlane(t, r * LANES);
      const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= row));
      b = l / LANES == r ? n : b;
    }
    const int to = b < c.batch ? b : 0; // (shuffles by every lane)
    const int e = __shfl(end, to, 64), len = __shfl(length, to, 64);
    if (!in || t < start || b >= c.batch)
      return RowPlace{-1, 0};
    return RowPlace{b, (int64_t)len - e + t};
  }
  const int b = in ? fhip_sequence_of(offsets, c.batch, t) : -1;
  return RowPlace{b, b < 0 ? 0 : (int64_t)c.lengths[b] - offsets[b + 1] + t};
}

// Extremes over the LANES lanes of a group.
template <bool MAX> __device__ __forceinline__ float extreme(float a, float b) { return MAX ? fmaxf(a, b) : fminf(a, b); }
template <bool MAX> __device__ __forceinline__ float over_group(float x, int lanes) {
  auto dpp = [](float v, auto ctrl) {
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  using std::integral_constant;
  x = extreme<MAX>(x, dpp(x, integral_constant<int, 0xb1>{})); // quad_perm 1 0 3 2
  x = extreme<MAX>(x, dpp(x, integral_constant<int, 0x4e>{})); // quad_perm 2 3 0 1
  if (lanes >= 8)
    x = extreme<MAX>(x, dpp(x, integral_constant<int, 0x141>{})); // row_half_mirror
  if (lanes >= 16)
    x = extreme<MAX>(x, dpp(x, integral_constant<int, 0x140>{})); // row_mirror
  if (lanes >= 32)
    x = extreme<MAX>(x, __shfl_xor(x, 16, 64));
  return x;
}

// 8 elements `at` of the row at (page, slot) of head h: `bits` as they are in 16 bits, their values in 4.
__device__ __forceinline__ void hold(const FhipCacheView &c, const FhipPool &p, int page, int slot, int h, int at,
                                     const u32x4 &bits, const float (&y)[8], bool in) {
  if (!c.group) {
    if (in)
      *(u32x4 *)(p.data + (page * p.page + h * p.head + slot * p.slot + at) * 2) = bits;
    return;
  }
  float lo = y[0], hi = y[0];
  bool number = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, y[i]), hi = fmaxf(hi, y[i]);
    number &= __builtin_fabsf(y[i]) < INFINITY;
  }
  hi = number ? hi : INFINITY; // (and so is the group's scale: none)
  const int lanes = c.group / 8;
  lo = over_group<false>(lo, lanes), hi = over_group<true>(hi, lanes);
  const FhipGroup g = fhip_group_of(lo, hi);
  const uint32_t codes = fhip_codes_of(g, y);
  if (!in)
    return;
  *(uint32_t *)(p.data + page * p.page + h * p.head + slot * p.slot + at / 2) = codes;
  if (at % c.group == 0) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    *(h2 *)(p.params + page * p.params_page + h * p.params_head + slot * p.params_slot + at / c.group * 2) = h2{g.scale, g.low};
  }
}

// LANES lanes per row (a power of two, D / 8 at least); N heads per wavefront.
template <bool BF16, int LANES, int N> __global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs g) {
#pragma clang fp contract(off)
  const int l = threadIdx.x & 63;
  const int t = (int)fhip_line_index(blockIdx.z) * (kThreads / LANES) + threadIdx.x / LANES, at = l % LANES * 8;
  const bool in = t < g.T;
  // heads of Q, of K, of V in slices of N
  const int q_slices = (g.Hq + N - 1) / N, k_slices = (g.Hkv + N - 1) / N;
  const int which = (int)blockIdx.y < q_slices ? 0 : (int)blockIdx.y < q_slices + k_slices ? 1 : 2;
  const int h0 = ((int)blockIdx.y - (which == 0 ? 0 : which == 1 ? q_slices : q_slices + k_slices)) * N;
  const int heads = which == 0 ? g.Hq : g.Hkv, D = which == 2 ? g.Dv : g.D, R = which == 2 ? 0 : g.R, half = R / 2;
  const char *x = (const char *)(which == 0 ? g.q : which == 1 ? g.k : g.v);
  const int64_t *xs = which == 0 ? g.q_s : which == 1 ? g.k_s : g.v_s;
  const bool mine = in && at < D;
  const bool turns = mine && at < R;
  const bool second = at >= half; // of a pair's elements, where halves are paired
  const int64_t row = (in ? t : 0) * xs[0];
  u32x4 own[N], other[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    own[i] = other[i] = u32x4{};
    if (mine && h0 + i < heads) {
      const char *from = x + (row + (h0 + i) * xs[1]) * 2;
      own[i] = *(const u32x4 *)(from + at * 2);
      if (turns && !g.interleaved)
        other[i] = *(const u32x4 *)(from + (second ? at - half : at + half) * 2);
    }
  }
  const int64_t given = g.positions && in ? g.positions[t] : 0;
  const RowPlace r = place_of<LANES>(g.cache, g.offsets, t, in);
  const int64_t pos = g.positions ? given : r.place;
  const bool turned = !g.R || (pos >= 0 && pos < g.table_rows);
  const int page = r.b >= 0 && which != 0 && r.place >= 0 && r.place < kCacheMaxKeys ? fhip_page_of(g.cache, r.b, (int)r.place) : -1;
  const int slot = page < 0 ? 0 : (int)((uint32_t)r.place % (uint32_t)g.cache.page_size);
  float c[8], s[8]; // (interleaved: four of each)
  if (R) {
    const bool load = turns && turned && r.b >= 0;
    const float *angles = g.rotation + (load ? pos * g.rot_s + (g.interleaved ? at / 2 : second ? at - half : at) : 0);
    f32x4 v[4] = {};
    if (load) {
      v[0] = *(const f32x4 *)angles, v[2] = *(const f32x4 *)(angles + half);
      if (!g.interleaved)
        v[1] = *(const f32x4 *)(angles + 4), v[3] = *(const f32x4 *)(angles + half + 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = v[i / 4][i % 4], s[i] = g.interleaved || second ? v[2 + i / 4][i % 4] : -v[2 + i / 4][i % 4];
  }
  void *out = which == 0 ? g.q_out : which == 1 ? g.k_out : nullptr;
  const int64_t *os = which == 0 ? g.qo_s : g.ko_s;
  const FhipPool &pool = which == 1 ? g.cache.k : g.cache.v;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (h0 + i >= heads) // (the wavefront's)
      break;
    float y[8];
    widen<BF16>(own[i], y);
    u32x4 bits = own[i];
    if (R) {
      if (turns) {
        float z[8];
        if (g.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float a = y[e] * c[e / 2], b = y[e + 1] * s[e / 2];
            const float d = y[e + 1] * c[e / 2], f = y[e] * s[e / 2];
            z[e] = a - b, z[e + 1] = d + f;
          }
        } else {
          float w[8];
          widen<BF16>(other[i], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = y[e] * c[e], b = w[e] * s[e]; // (the first element's sine has its sign)
            z[e] = a + b;
          }
        }
        bits = narrow<BF16>(z);
      }
      if (!turned)
        bits = BF16 ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}
                    : u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
      if (which != 0)
        widen<BF16>(bits, y);
    }
    if (out && mine && r.b >= 0)
      *(u32x4 *)((char *)out + (t * os[0] + (h0 + i) * os[1] + at) * 2) = bits;
    if (which != 0)
      hold(g.cache, pool, page < 0 ? 0 : page, slot, h0 + i, at, bits, y, mine && page >= 0 && turned);
  }
}

template <bool BF16, int LANES, int N> __global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs g) {
#pragma clang fp contract(off)
  const int l = threadIdx.x & 63;
  const int t = (int)fhip_line_index(blockIdx.z) * (kThreads / LANES) + threadIdx.x / LANES, at = l % LANES * 8;
  const bool in = t < g.T;
  const int slices = (g.Hkv + N - 1) / N;
  const RowPlace r = place_of<LANES>(g.cache, g.offsets, t, in);
  const int page = r.b >= 0 && r.place >= 0 && r.place < kCacheMaxKeys ? fhip_page_of(g.cache, r.b, (int)r.place) : -1;
  const int slot = page < 0 ? 0 : (int)((uint32_t)r.place % (uint32_t)g.cache.page_size);
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  for (int slice = blockIdx.y; slice < 2 * slices; slice += gridDim.y) {
    const bool is_k = slice < slices;
    const int h0 = (slice - (is_k ? 0 : slices)) * N, D = is_k ? g.D : g.Dv;
    const FhipPool &p = is_k ? g.cache.k : g.cache.v;
    const bool mine = in && at < D && r.b >= 0, load = mine && page >= 0;
    const int64_t from = page < 0 ? 0 : page * p.page + slot * p.slot, pair = page < 0 ? 0 : page * p.params_page + slot * p.params_slot;
    char *out = (char *)(is_k ? g.k : g.v) + (t * (is_k ? g.k_s[0] : g.v_s[0]) + at) * 2;
    const int64_t out_h = is_k ? g.k_s[1] : g.v_s[1];
    u32x4 bits[N];
    h2 scale[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      bits[i] = BF16 ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}
                     : u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
      if (load && h0 + i < g.Hkv) {
        const int64_t row = from + (h0 + i) * p.head;
        if (g.cache.group) {
          bits[i].x = *(const uint32_t *)(p.data + row + at / 2);
          scale[i] = *(const h2 *)(p.params + pair + (h0 + i) * p.params_head + at / g.cache.group * 2);
        } else {
          bits[i] = *(const u32x4 *)(p.data + (row + at) * 2);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (g.cache.group && load) {
        const uint32_t w = bits[i].x;
        const float a = (float)scale[i].x, b = (float)scale[i].y;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = b + a * (float)(w >> (4 * e) & 15); // (the product is exact)
        bits[i] = narrow<BF16>(y);
      }
      if (mine && h0 + i < g.Hkv)
        *(u32x4 *)(out + (h0 + i) * out_h * 2) = bits[i];
    }
  }
}

// Whether strides of all dims but the last, and the start, are on `step` elements.
bool fits(const fhip_tensor_desc &t, int64_t step) {
  for (int i = 0; i + 1 < t.rank; ++i)
    if (t.dim[i] > 1 && t.stride[i] % step != 0)
      return false;
  return true;
}
bool cache_fits(const fhip_cache_desc &c, int64_t D, int64_t Dv) {
  if (D % 8 != 0 || Dv % 8 != 0)
    return false;
  if (c.k_params.rank == 0)
    return fits(c.k, 8) && fits(c.v, 8);
  const int64_t group = 2 * D / c.k_params.dim[3];
  return (group == 32 || group == 64 || group == 128 || group == 256) && fits(c.k, 4) && fits(c.v, 4) &&
         fits(c.k_params, 2) && fits(c.v_params, 2);
}
bool cache_aligned(const fhip_cache_desc &c, const fhip_cache_ptrs &p) {
  const uintptr_t data = (uintptr_t)p.k | (uintptr_t)p.v, pairs = (uintptr_t)p.k_params | (uintptr_t)p.v_params;
  return (data & (c.k_params.rank ? 3 : 15)) == 0 && (pairs & 3) == 0;
}
bool append_fits(const fhip_cache_append_desc &d) {
  const int dt = d.k.dtype;
  if ((dt != FHIP_BFLOAT16 && dt != FHIP_HALF) || !cache_fits(d.cache, d.k.dim[2], d.v.dim[2]))
    return false;
  if (!fits(d.k, 8) || !fits(d.v, 8) || !fits(d.q, 8) || !fits(d.q_out, 8) || !fits(d.k_out, 8))
    return false;
  return d.rotation.rank == 0 || (d.rotation.dim[1] % 16 == 0 && fits(d.rotation, 4));
}
bool read_fits(const fhip_cache_read_desc &d) {
  const int dt = d.k.dtype;
  return (dt == FHIP_BFLOAT16 || dt == FHIP_HALF) && cache_fits(d.cache, d.k.dim[2], d.v.dim[2]) && fits(d.k, 8) &&
         fits(d.v, 8);
}
// go(type, lanes, heads) as constants.
template <typename F> int with_lanes(bool bf16, int lanes, int heads, F &&go) {
  using std::integral_constant;
  auto headed = [&](auto bf, auto lc) {
    return heads == 4 ? go(bf, lc, integral_constant<int, 4>{}) : go(bf, lc, integral_constant<int, 1>{});
  };
  auto sized = [&](auto bf) {
    return lanes == 8    ? headed(bf, integral_constant<int, 8>{})
           : lanes == 16 ? headed(bf, integral_constant<int, 16>{})
           : lanes == 32 ? headed(bf, integral_constant<int, 32>{})
                         : headed(bf, integral_constant<int, 64>{});
  };
  return bf16 ? sized(std::true_type{}) : sized(std::false_type{});
}
// Lanes of a row of 8 * chunks elements.
int lanes_of(int64_t D, int64_t Dv) {
  const int64_t most = D > Dv ? D : Dv;
  return most <= 64 ? 8 : most <= 128 ? 16 : most <= 256 ? 32 : 64;
}

// Whether every element of both lies at the same offset.
bool same_tensor(const fhip_tensor_desc &a, const fhip_tensor_desc &b) {
  for (int i = 0; i < a.rank; ++i)
    if (a.dim[i] > 1 && a.stride[i] != b.stride[i])
      return false;
  return a.dtype == b.dtype;
}

} // namespace

FhipCacheView fhip_cache_view(const fhip_cache_desc &c, const fhip_cache_ptrs &p) {
  FhipCacheView w{};
  auto pool = [&](const fhip_tensor_desc &t, const fhip_tensor_desc &pt, void *data, void *params) {
    auto st = [](const fhip_tensor_desc &x, int i) { return x.dim[i] > 1 ? x.stride[i] : 0; };
    FhipPool o{(char *)data, (_Float16 *)params, st(t, 0), st(t, 1), st(t, 2), 0, 0, 0};
    if (pt.rank)
      o.params_page = st(pt, 0), o.params_head = st(pt, 1), o.params_slot = st(pt, 2);
    return o;
  };
  w.k = pool(c.k, c.k_params, p.k, p.k_params);
  w.v = pool(c.v, c.v_params, p.v, p.v_params);
  w.table = (const int32_t *)p.pages;
  w.lengths = (const int32_t *)p.lengths;
  w.table_stride = c.batch > 1 ? c.page_stride : 0;
  w.batch = (int32_t)c.batch;
  w.table_pages = (int32_t)c.pages_per_sequence;
  w.pool_pages = (int32_t)c.k.dim[0];
  w.page_size = (int32_t)c.k.dim[2];
  w.group = c.k_params.rank ? (int32_t)(2 * c.k.dim[3] / (c.k_params.dim[3] / 2)) : 0;
  w.dtype = c.k.dtype;
  return w;
}

int fhip_check_rows(fhip_ctx *ctx, const char *who, const char *what, const fhip_tensor_desc &t, bool written) {
  if (!fhip_check_desc(ctx, t, what))
    return 1;
  FHIP_REQUIRE(ctx, t.rank == 3, "%s: %s must be rank 3 [rows, heads, head dim]", who, what);
  FHIP_REQUIRE(ctx, t.dtype == FHIP_FLOAT || t.dtype == FHIP_BFLOAT16 || t.dtype == FHIP_HALF,
               "%s: %s must be f32, bf16 or f16", who, what);
  FHIP_REQUIRE(ctx, t.dim[0] < (1ll << 31) - 1 && t.dim[1] < (1 << 20) && t.dim[2] <= kCacheMaxDim,
               "%s: %s has rows, heads or a head dim (above %d) out of range", who, what, kCacheMaxDim);
  FHIP_REQUIRE(ctx, t.dim[2] == 1 || t.stride[2] == 1, "%s: %s must have a unit stride in its last dim", who, what);
  FHIP_REQUIRE(ctx, !written || ((t.dim[0] == 1 || t.stride[0] > 0) && (t.dim[1] == 1 || t.stride[1] > 0)),
               "%s: %s is written and has a stride of 0", who, what);
  return 0;
}

int fhip_check_cache(fhip_ctx *ctx, const char *who, const fhip_cache_desc &c, int dtype, int64_t heads, int64_t D,
                     int64_t Dv) {
  if (!fhip_check_desc(ctx, c.k, "cache K") || !fhip_check_desc(ctx, c.v, "cache V"))
    return 1;
  FHIP_REQUIRE(ctx, c.k.rank == 4 && c.v.rank == 4,
               "%s: the cache's K and V must be rank 4 [pages, heads, page size, head dim]", who);
  for (int i = 0; i < 3; ++i)
    FHIP_REQUIRE(ctx, c.k.dim[i] == c.v.dim[i], "%s: the cache's K and V differ in dim %d", who, i);
  FHIP_REQUIRE(ctx, c.k.dim[0] < (1ll << 31) && c.k.dim[2] <= (1 << 24), "%s: pages or page size out of range", who);
  FHIP_REQUIRE(ctx, c.k.dim[1] == heads, "%s: the cache has %lld heads, the rows %lld", who, (long long)c.k.dim[1],
               (long long)heads);
  FHIP_REQUIRE(ctx, c.k.dtype == c.v.dtype, "%s: the cache's K and V differ in type", who);
  const bool packed = c.k.dtype == FHIP_UINT8;
  FHIP_REQUIRE(ctx, packed || c.k.dtype == dtype, "%s: the cache must have the rows' type, or be Uint8 with parameters",
               who);
  FHIP_REQUIRE(ctx, packed == (c.k_params.rank != 0) && packed == (c.v_params.rank != 0),
               "%s: parameters go with a Uint8 cache, and only with one", who);
  const int64_t div = packed ? 2 : 1;
  FHIP_REQUIRE(ctx, D % div == 0 && Dv % div == 0 && c.k.dim[3] == D / div && c.v.dim[3] == Dv / div,
               "%s: the cache's head dims do not fit the rows'", who);
  const fhip_tensor_desc *ts[4] = {&c.k, &c.v, &c.k_params, &c.v_params};
  for (int i = 0; i < (packed ? 4 : 2); ++i) {
    const fhip_tensor_desc &t = *ts[i];
    if (i >= 2) {
      if (!fhip_check_desc(ctx, t, "cache parameters"))
        return 1;
      FHIP_REQUIRE(ctx, t.rank == 4 && t.dtype == FHIP_HALF && t.dim[0] == c.k.dim[0] && t.dim[1] == heads &&
                            t.dim[2] == c.k.dim[2],
                   "%s: the cache's parameters must be Half [pages, heads, page size, pairs]", who);
    }
    FHIP_REQUIRE(ctx, t.dim[3] == 1 || t.stride[3] == 1, "%s: the cache needs a unit stride in its last dim", who);
    for (int j = 0; j < 3; ++j)
      FHIP_REQUIRE(ctx, t.dim[j] == 1 || t.stride[j] > 0, "%s: the cache has a stride of 0", who);
  }
  if (packed) {
    const int64_t nk = c.k_params.dim[3] / 2, nv = c.v_params.dim[3] / 2;
    FHIP_REQUIRE(ctx, c.k_params.dim[3] % 2 == 0 && c.v_params.dim[3] % 2 == 0 && nk > 0 && nv > 0 && D % nk == 0 &&
                          Dv % nv == 0 && D / nk % 2 == 0 && D / nk == Dv / nv,
                 "%s: groups must be of an even number of elements that divides the head dims, the same for K and V",
                 who);
  }
  FHIP_REQUIRE(ctx, c.batch >= 1 && c.batch < (1 << 30), "%s: batch %lld out of range", who, (long long)c.batch);
  FHIP_REQUIRE(ctx, c.pages_per_sequence >= 1 && c.pages_per_sequence < (1ll << 31) &&
                        c.pages_per_sequence * c.k.dim[2] <= kCacheMaxKeys,
               "%s: the page table holds more than 2^30 keys per sequence, or none", who);
  FHIP_REQUIRE(ctx, c.batch == 1 || c.page_stride >= c.pages_per_sequence, "%s: the page table's rows overlap", who);
  return 0;
}

int fhip_check_cache_ptrs(fhip_ctx *ctx, const char *who, const fhip_cache_desc &c, const fhip_cache_ptrs *p) {
  FHIP_REQUIRE(ctx, p && p->k && p->v && p->pages && p->lengths, "%s: null cache pointer", who);
  FHIP_REQUIRE(ctx, (c.k_params.rank != 0) == (p->k_params != nullptr) &&
                        (c.v_params.rank != 0) == (p->v_params != nullptr),
               "%s: parameter pointers and descriptors disagree", who);
  return 0;
}

static int append_validate(fhip_ctx *ctx, const fhip_cache_append_desc *d) {
  static const char who[] = "fhip_cache_append";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (fhip_check_rows(ctx, who, "K", d->k, false) || fhip_check_rows(ctx, who, "V", d->v, false))
    return 1;
  const int64_t T = d->k.dim[0], Hkv = d->k.dim[1], D = d->k.dim[2], Dv = d->v.dim[2];
  FHIP_REQUIRE(ctx, d->v.dim[0] == T && d->v.dim[1] == Hkv && d->v.dtype == d->k.dtype,
               "%s: K and V differ in rows, heads or type", who);
  FHIP_REQUIRE(ctx, (d->q.rank != 0) == (d->q_out.rank != 0), "%s: Q and Q_OUT go together", who);
  if (d->q.rank) {
    if (fhip_check_rows(ctx, who, "Q", d->q, false) || fhip_check_rows(ctx, who, "Q_OUT", d->q_out, true))
      return 1;
    for (int i = 0; i < 3; ++i)
      FHIP_REQUIRE(ctx, d->q.dim[i] == d->q_out.dim[i], "%s: Q_OUT dims differ from Q's", who);
    FHIP_REQUIRE(ctx, d->q.dim[0] == T && d->q.dim[2] == D && d->q.dtype == d->k.dtype && d->q_out.dtype == d->k.dtype,
                 "%s: Q, Q_OUT and K differ in rows, head dim or type", who);
  }
  if (d->k_out.rank) {
    if (fhip_check_rows(ctx, who, "K_OUT", d->k_out, true))
      return 1;
    for (int i = 0; i < 3; ++i)
      FHIP_REQUIRE(ctx, d->k.dim[i] == d->k_out.dim[i], "%s: K_OUT dims differ from K's", who);
    FHIP_REQUIRE(ctx, d->k_out.dtype == d->k.dtype, "%s: K_OUT has another type than K", who);
  }
  if (d->rotation.rank) {
    const fhip_tensor_desc &r = d->rotation;
    if (!fhip_check_desc(ctx, r, "ROTATION"))
      return 1;
    FHIP_REQUIRE(ctx, r.rank == 2 && r.dtype == FHIP_FLOAT && r.stride[1] == 1 && r.dim[0] < (1ll << 31),
                 "%s: ROTATION must be Float [positions, R] with a unit stride in its last dim", who);
    FHIP_REQUIRE(ctx, r.dim[1] % 2 == 0 && r.dim[1] <= D, "%s: ROTATION turns %lld of %lld dims", who,
                 (long long)r.dim[1], (long long)D);
  }
  const int64_t heads = (d->q.rank ? d->q.dim[1] : 0) + 2 * Hkv;
  FHIP_REQUIRE(ctx, T * heads < (1ll << 31), "%s: more than 2^31 rows of heads", who);
  return fhip_check_cache(ctx, who, d->cache, d->k.dtype, Hkv, D, Dv);
}

static int read_validate(fhip_ctx *ctx, const fhip_cache_read_desc *d) {
  static const char who[] = "fhip_cache_read";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (fhip_check_rows(ctx, who, "K", d->k, true) || fhip_check_rows(ctx, who, "V", d->v, true))
    return 1;
  FHIP_REQUIRE(ctx, d->v.dim[0] == d->k.dim[0] && d->v.dim[1] == d->k.dim[1] && d->v.dtype == d->k.dtype,
               "%s: K and V differ in rows, heads or type", who);
  FHIP_REQUIRE(ctx, d->k.dim[0] * d->k.dim[1] < (1ll << 30), "%s: more than 2^30 rows of heads", who);
  return fhip_check_cache(ctx, who, d->cache, d->k.dtype, d->k.dim[1], d->k.dim[2], d->v.dim[2]);
}

extern "C" {

int fhip_cache_append_workspace_size(const fhip_cache_append_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_cache_append_workspace_size: null");
  *bytes = 0;
  return 0;
}

int fhip_cache_append_supported(const fhip_cache_append_desc *d) {
  if (!d || append_validate(nullptr, d) != 0)
    return 0;
  return append_fits(*d) ? 2 : 1;
}

int fhip_cache_append(fhip_ctx *ctx, const fhip_cache_append_desc *d, const fhip_cache_ptrs *cache, const void *q,
                      const void *k, const void *v, const void *rotation, const void *offsets, const void *positions,
                      void *q_out, void *k_out, void *workspace, size_t workspace_bytes) {
  static const char who[] = "fhip_cache_append";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (append_validate(ctx, d) != 0 || fhip_check_cache_ptrs(ctx, who, d->cache, cache) != 0)
    return 1;
  FHIP_REQUIRE(ctx, k && v && offsets, "%s: null tensor pointer", who);
  FHIP_REQUIRE(ctx, (d->q.rank != 0) == (q != nullptr) && (d->q.rank != 0) == (q_out != nullptr),
               "%s: Q / Q_OUT pointers and descriptors disagree", who);
  FHIP_REQUIRE(ctx, (d->k_out.rank != 0) == (k_out != nullptr), "%s: K_OUT pointer and descriptor disagree", who);
  FHIP_REQUIRE(ctx, (d->rotation.rank != 0) == (rotation != nullptr), "%s: ROTATION pointer and descriptor disagree",
               who);
  FHIP_REQUIRE(ctx, (d->has_positions != 0) == (positions != nullptr), "%s: positions and has_positions disagree", who);
  FHIP_REQUIRE(ctx, (q_out != q || same_tensor(d->q, d->q_out)) && (k_out != k || same_tensor(d->k, d->k_out)),
               "%s: a row that is turned in place needs the same strides", who);
  (void)workspace;
  (void)workspace_bytes;
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  AppendArgs g{};
  g.q = q, g.k = k, g.v = v, g.q_out = q_out, g.k_out = k_out;
  g.rotation = (const float *)rotation;
  g.offsets = (const int32_t *)offsets, g.positions = (const int32_t *)positions;
  g.cache = fhip_cache_view(d->cache, *cache);
  auto st = [](const fhip_tensor_desc &t, int64_t(&s)[2]) { s[0] = t.stride[0], s[1] = t.stride[1]; };
  st(d->q, g.q_s), st(d->k, g.k_s), st(d->v, g.v_s), st(d->q_out, g.qo_s), st(d->k_out, g.ko_s);
  g.dtype = d->k.dtype;
  g.T = (int32_t)d->k.dim[0], g.Hq = d->q.rank ? (int32_t)d->q.dim[1] : 0, g.Hkv = (int32_t)d->k.dim[1];
  g.D = (int32_t)d->k.dim[2], g.Dv = (int32_t)d->v.dim[2];
  if (d->rotation.rank)
    g.R = (int32_t)d->rotation.dim[1], g.table_rows = (int32_t)d->rotation.dim[0], g.rot_s = d->rotation.stride[0];
  g.interleaved = d->interleaved != 0;
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)rotation | (uintptr_t)q_out | (uintptr_t)k_out;
  if (append_fits(*d) && (all & 15) == 0 && cache_aligned(d->cache, *cache)) {
    const int lanes = lanes_of(g.D, g.Dv);
    const int64_t rows = kThreads / lanes, blocks = (g.T + rows - 1) / rows;
    // heads of a wavefront: four, where a thousand workgroups are left
    const int n = blocks * ((g.Hq + 3) / 4 + 2 * ((g.Hkv + 3) / 4)) >= 1024 ? 4 : 1;
    const int64_t slices = (g.Hq + n - 1) / n + 2 * (int64_t)((g.Hkv + n - 1) / n);
    if (slices <= 65535) {
      fhip_note_kernel(ctx, "cache_append bits=%d lanes=%d heads=%d", d->cache.k_params.rank ? 4 : 16, lanes, n);
      return with_lanes(d->k.dtype == FHIP_BFLOAT16, lanes, n, [&](auto bf, auto lc, auto nc) {
        hipLaunchKernelGGL((append_kernel<decltype(bf)::value, decltype(lc)::value, decltype(nc)::value>),
                           fhip_line_grid(blocks, (unsigned)slices), dim3(kThreads), 0, ctx->stream, g);
        FHIP_HIP_CHECK(ctx, hipGetLastError());
        return 0;
      });
    }
  }
  fhip_note_kernel(ctx, "cache_append_rows");
  hipLaunchKernelGGL(append_rows_kernel, fhip_line_grid((int64_t)g.T * (g.Hq + 2 * g.Hkv)), dim3(64), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

int fhip_cache_read_workspace_size(const fhip_cache_read_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_cache_read_workspace_size: null");
  *bytes = 0;
  return 0;
}

int fhip_cache_read_supported(const fhip_cache_read_desc *d) {
  if (!d || read_validate(nullptr, d) != 0)
    return 0;
  return read_fits(*d) ? 2 : 1;
}

int fhip_cache_read(fhip_ctx *ctx, const fhip_cache_read_desc *d, const fhip_cache_ptrs *cache, const void *offsets,
                    void *k, void *v, void *workspace, size_t workspace_bytes) {
  static const char who[] = "fhip_cache_read";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (read_validate(ctx, d) != 0 || fhip_check_cache_ptrs(ctx, who, d->cache, cache) != 0)
    return 1;
  FHIP_REQUIRE(ctx, k && v && offsets, "%s: null tensor pointer", who);
  (void)workspace;
  (void)workspace_bytes;
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  ReadArgs g{};
  g.k = k, g.v = v, g.offsets = (const int32_t *)offsets;
  g.cache = fhip_cache_view(d->cache, *cache);
  g.k_s[0] = d->k.stride[0], g.k_s[1] = d->k.stride[1], g.v_s[0] = d->v.stride[0], g.v_s[1] = d->v.stride[1];
  g.dtype = d->k.dtype;
  g.T = (int32_t)d->k.dim[0], g.Hkv = (int32_t)d->k.dim[1], g.D = (int32_t)d->k.dim[2], g.Dv = (int32_t)d->v.dim[2];
  if (read_fits(*d) && (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && cache_aligned(d->cache, *cache)) {
    const int lanes = lanes_of(g.D, g.Dv);
    const int64_t rows = kThreads / lanes, blocks = (g.T + rows - 1) / rows;
    const int n = blocks * 2 * ((g.Hkv + 3) / 4) >= 1024 ? 4 : 1;
    const int64_t slices = 2 * (int64_t)((g.Hkv + n - 1) / n);
    // a workgroup takes slices in turn, each behind the one search for its rows' pages, where a thousand workgroups
    // are left: 26656 rows of 8 heads out of 4 bits 33.6 us with one workgroup for all, 36.0 with two, 39.0 with four
    const int64_t beside = blocks >= 1024 ? 1 : blocks * slices <= 1024 ? slices : (1024 + blocks - 1) / blocks;
    if (slices <= 65535) {
      fhip_note_kernel(ctx, "cache_read bits=%d lanes=%d heads=%d", d->cache.k_params.rank ? 4 : 16, lanes, n);
      return with_lanes(d->k.dtype == FHIP_BFLOAT16, lanes, n, [&](auto bf, auto lc, auto nc) {
        hipLaunchKernelGGL((read_kernel<decltype(bf)::value, decltype(lc)::value, decltype(nc)::value>),
                           fhip_line_grid(blocks, (unsigned)beside), dim3(kThreads), 0, ctx->stream, g);
        FHIP_HIP_CHECK(ctx, hipGetLastError());
        return 0;
      });
    }
  }
  fhip_note_kernel(ctx, "cache_read_rows");
  hipLaunchKernelGGL(read_rows_kernel, fhip_line_grid((int64_t)g.T * 2 * g.Hkv), dim3(64), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
