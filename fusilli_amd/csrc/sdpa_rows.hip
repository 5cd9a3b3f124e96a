// Attention of packed sequences, on each other or over a cache in pages: the
// entry points, and the kernel for any type, size, stride and page size: one to
// eight wavefronts per row of one query head, each with every so many blocks of 64 keys.
//
//   O[r] = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),  s_j = scale Q[r] . K_j,
// over the keys that row r sees; the running maximum m and sum in f32.
//
// Bound by its element loads: a lane walks a key of its own, then the wavefront
// walks the keys together, a column per lane.  Head dim 80, bf16, 32 heads on 8:
// 32 tokens over 86347 keys 2.7 ms (one wavefront per row: 11.7), 24 prompts of
// 16 to 512 tokens 6.7 ms.
#include "paged_cache.h"
#include "fast_paths.h"

#include <cmath>

namespace {

struct RowsArgs {
  const void *q, *k, *v; // k, v null: the cache
  void *o;
  const int32_t *offsets, *kv_offsets;
  FhipCacheView cache;
  int64_t q_s[2], k_s[2], v_s[2], o_s[2];
  int32_t dtype, batch, T, Tk, Hq, group, D, Dv, causal;
  float scale;
};

constexpr int kPerLane = kCacheMaxDim / 64;

__device__ __forceinline__ float wave_reduce(float x, bool max) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float y = __shfl_xor(x, o, 64);
    x = max ? fmaxf(x, y) : x + y;
  }
  return x;
}

constexpr int kRowWaves = 8;

__global__ __launch_bounds__(64 * kRowWaves) void sdpa_rows_kernel(RowsArgs g) {
  extern __shared__ float query[]; // [D], then for each wavefront its maximum and sum, and [Dv] parts
  const uint32_t line = fhip_line_index(blockIdx.y);
  const int t = (int)(line / (uint32_t)g.Hq), h = (int)(line % (uint32_t)g.Hq), hk = h / g.group;
  if (t >= g.T)
    return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  float *const tops = query + g.D, *const sums = tops + waves, *const part = sums + waves;
  const int b = fhip_sequence_of(g.offsets, g.batch, t);
  if (b < 0)
    return;
  const int64_t behind = (int64_t)g.offsets[b + 1] - t; // rows of the sequence from this one on
  int64_t first = 0, keys; // the sequence's keys; the first one's packed row
  int64_t stored; // keys that the page table has places for
  if (g.k) {
    const int64_t a = g.kv_offsets[b], e = g.kv_offsets[b + 1];
    first = a < 0 ? 0 : a > g.Tk ? g.Tk : a;
    keys = (e > g.Tk ? g.Tk : e) - first;
    stored = keys;
  } else {
    keys = g.cache.lengths[b];
    stored = (int64_t)g.cache.table_pages * g.cache.page_size;
  }
  int64_t seen = g.causal ? keys - behind + 1 : keys;
  bool bad = seen > stored;
  seen = seen < 0 ? 0 : bad ? stored : seen;
  for (int e = threadIdx.x; e < g.D; e += blockDim.x)
    query[e] = fhip_load<float>(g.q, g.dtype, t * g.q_s[0] + h * g.q_s[1] + e);
  __syncthreads();
  float acc[kPerLane];
  for (int e = 0; e < kPerLane; ++e)
    acc[e] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int64_t j0 = wave * 64; j0 < seen; j0 += waves * 64) {
    const int64_t j = j0 + lane;
    float s = -INFINITY;
    if (j < seen) {
      float dot = 0.f;
      if (g.k) {
        const int64_t at = (first + j) * g.k_s[0] + hk * g.k_s[1];
        for (int e = 0; e < g.D; ++e)
          dot += query[e] * fhip_load<float>(g.k, g.dtype, at + e);
      } else {
        const int page = fhip_page_of(g.cache, b, (int)j);
        if (page < 0)
          dot = __builtin_nanf("");
        else
          for (int e = 0; e < g.D; ++e)
            dot += query[e] * fhip_cache_value(g.cache, g.cache.k, page, (int)(j % g.cache.page_size), hk, e);
      }
      s = dot * g.scale;
    }
    bad |= __builtin_amdgcn_ballot_w64(s != s) != 0;
    // (a NaN score is not above the maximum; it makes the whole row NaN below)
    const float m_new = fmaxf(m, wave_reduce(s, true));
    const float p = m_new == -INFINITY ? 0.f : __expf(s - m_new);
    const float fade = m_new == -INFINITY ? 1.f : __expf(m - m_new);
    l = l * fade + wave_reduce(p, false);
    m = m_new;
    const int count = seen - j0 < 64 ? (int)(seen - j0) : 64;
    for (int e = 0; e < kPerLane; ++e)
      acc[e] *= fade;
    for (int jj = 0; jj < count; ++jj) {
      const int page = g.k ? 0 : fhip_page_of(g.cache, b, (int)(j0 + jj));
      if (page < 0)
        continue;
      const float prob = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), jj));
      for (int e = 0; e < kPerLane; ++e) {
        const int d = lane + 64 * e;
        if (d >= g.Dv)
          break;
        acc[e] += prob * (g.k ? fhip_load<float>(g.v, g.dtype, (first + j0 + jj) * g.v_s[0] + hk * g.v_s[1] + d)
                                  : fhip_cache_value(g.cache, g.cache.v, page,
                                                     (int)((j0 + jj) % g.cache.page_size), hk, d));
      }
    }
  }
  // the wavefronts' parts meet (a wavefront without keys has the maximum -inf)
  for (int e = 0; e < kPerLane; ++e)
    if (lane + 64 * e < g.Dv)
      part[wave * g.Dv + lane + 64 * e] = acc[e];
  if (lane == 0)
    tops[wave] = m, sums[wave] = bad ? __builtin_nanf("") : l;
  __syncthreads();
  for (int w = 0; w < waves; ++w)
    m = fmaxf(m, tops[w]);
  for (int d = threadIdx.x; d < g.Dv; d += blockDim.x) {
    float sum = 0.f, den = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float f = tops[w] == -INFINITY ? 0.f : __expf(tops[w] - m);
      den += sums[w] == sums[w] ? sums[w] * f : sums[w];
      sum += part[w * g.Dv + d] * f;
    }
    fhip_store<float>(g.o, g.dtype, t * g.o_s[0] + h * g.o_s[1] + d,
                      den != den ? den : seen > 0 ? sum / den : 0.f);
  }
}

int launch_rows(fhip_ctx *ctx, RowsArgs &g, const fhip_tensor_desc &q, const fhip_tensor_desc &o, int64_t Hkv,
                bool has_scale, float scale) {
  g.q_s[0] = q.stride[0], g.q_s[1] = q.stride[1], g.o_s[0] = o.stride[0], g.o_s[1] = o.stride[1];
  g.dtype = q.dtype;
  g.T = (int32_t)q.dim[0], g.Hq = (int32_t)q.dim[1], g.D = (int32_t)q.dim[2], g.Dv = (int32_t)o.dim[2];
  g.group = (int32_t)(q.dim[1] / Hkv);
  g.scale = has_scale ? scale : 1.0f / sqrtf((float)g.D);
  // wavefronts that the rows leave idle share them: eight thousand fill the chip
  const int64_t rows = (int64_t)g.T * g.Hq;
  int waves = 1;
  while (waves < kRowWaves && rows * waves * 2 <= 8192)
    waves *= 2;
  hipLaunchKernelGGL(sdpa_rows_kernel, fhip_line_grid(rows), dim3(64 * waves),
                     sizeof(float) * (g.D + waves * (g.Dv + 2)), ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // namespace

static int check_q_o(fhip_ctx *ctx, const char *who, const fhip_tensor_desc &q, const fhip_tensor_desc &o,
                     int64_t Hkv, int64_t Dv) {
  FHIP_REQUIRE(ctx, q.dim[1] % Hkv == 0, "%s: %lld query heads are no multiple of %lld key heads", who,
               (long long)q.dim[1], (long long)Hkv);
  FHIP_REQUIRE(ctx, o.dim[0] == q.dim[0] && o.dim[1] == q.dim[1] && o.dim[2] == Dv && o.dtype == q.dtype,
               "%s: O must be [rows, query heads, value head dim] of Q's type", who);
  FHIP_REQUIRE(ctx, q.dim[0] * q.dim[1] < (1ll << 31), "%s: more than 2^31 rows of heads", who);
  return 0;
}

static int check_workspace(fhip_ctx *ctx, const char *who, size_t need, const void *workspace, size_t bytes) {
  FHIP_REQUIRE(ctx, need == 0 || (workspace && bytes >= need && ((uintptr_t)workspace & 255) == 0),
               "%s: needs %zu bytes of 256-byte aligned workspace, got %zu", who, need, bytes);
  return 0;
}

static int packed_validate(fhip_ctx *ctx, const fhip_sdpa_packed_desc *d) {
  static const char who[] = "fhip_sdpa_packed_fwd";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (fhip_check_rows(ctx, who, "Q", d->q, false) || fhip_check_rows(ctx, who, "K", d->k, false) ||
      fhip_check_rows(ctx, who, "V", d->v, false) || fhip_check_rows(ctx, who, "O", d->o, true))
    return 1;
  FHIP_REQUIRE(ctx, d->k.dtype == d->q.dtype && d->v.dtype == d->q.dtype, "%s: Q, K and V differ in type", who);
  FHIP_REQUIRE(ctx, d->k.dim[2] == d->q.dim[2], "%s: Q/K head dim mismatch", who);
  FHIP_REQUIRE(ctx, d->v.dim[0] == d->k.dim[0] && d->v.dim[1] == d->k.dim[1], "%s: K and V differ in rows or heads",
               who);
  FHIP_REQUIRE(ctx, d->has_kv_offsets || d->k.dim[0] == d->q.dim[0], "%s: without kv_offsets K has Q's rows", who);
  FHIP_REQUIRE(ctx, d->batch >= 1 && d->batch < (1 << 30), "%s: batch %lld out of range", who, (long long)d->batch);
  return check_q_o(ctx, who, d->q, d->o, d->k.dim[1], d->v.dim[2]);
}

static int paged_validate(fhip_ctx *ctx, const fhip_sdpa_paged_desc *d) {
  static const char who[] = "fhip_sdpa_paged_fwd";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (fhip_check_rows(ctx, who, "Q", d->q, false) || fhip_check_rows(ctx, who, "O", d->o, true) ||
      !fhip_check_desc(ctx, d->cache.k, "cache K"))
    return 1;
  if (fhip_check_cache(ctx, who, d->cache, d->q.dtype, d->cache.k.dim[1], d->q.dim[2], d->o.dim[2]))
    return 1;
  return check_q_o(ctx, who, d->q, d->o, d->cache.k.dim[1], d->o.dim[2]);
}

extern "C" {

int fhip_sdpa_packed_fwd_workspace_size(const fhip_sdpa_packed_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_sdpa_packed_fwd_workspace_size: null");
  *bytes = 0;
  if (packed_validate(nullptr, d) != 0)
    return 1;
  if (fhip_fast_sdpa_packed_applicable(d))
    *bytes = fhip_fast_sdpa_packed_workspace(d);
  return 0;
}

int fhip_sdpa_packed_fwd_supported(const fhip_sdpa_packed_desc *d) {
  if (!d || packed_validate(nullptr, d) != 0)
    return 0;
  return fhip_fast_sdpa_packed_applicable(d) ? 2 : 1;
}

int fhip_sdpa_packed_fwd(fhip_ctx *ctx, const fhip_sdpa_packed_desc *d, const void *q, const void *k, const void *v,
                         const void *offsets, const void *kv_offsets, void *o, void *workspace,
                         size_t workspace_bytes) {
  static const char who[] = "fhip_sdpa_packed_fwd";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (packed_validate(ctx, d) != 0)
    return 1;
  FHIP_REQUIRE(ctx, q && k && v && offsets && o, "%s: null tensor pointer", who);
  FHIP_REQUIRE(ctx, (d->has_kv_offsets != 0) == (kv_offsets != nullptr), "%s: kv_offsets and has_kv_offsets disagree",
               who);
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  if (fhip_fast_sdpa_packed_applicable(d)) {
    if (check_workspace(ctx, who, fhip_fast_sdpa_packed_workspace(d), workspace, workspace_bytes))
      return 1;
    bool handled = false;
    const int rc = fhip_fast_sdpa_packed(ctx, d, q, k, v, offsets, kv_offsets, o, workspace, &handled);
    if (handled)
      return rc;
  }
  fhip_note_kernel(ctx, "sdpa_rows packed");
  RowsArgs g{};
  g.q = q, g.k = k, g.v = v, g.o = o;
  g.offsets = (const int32_t *)offsets, g.kv_offsets = (const int32_t *)(kv_offsets ? kv_offsets : offsets);
  g.k_s[0] = d->k.stride[0], g.k_s[1] = d->k.stride[1], g.v_s[0] = d->v.stride[0], g.v_s[1] = d->v.stride[1];
  g.batch = (int32_t)d->batch, g.Tk = (int32_t)d->k.dim[0], g.causal = d->is_causal != 0;
  return launch_rows(ctx, g, d->q, d->o, d->k.dim[1], d->has_scale, d->scale);
}

int fhip_sdpa_paged_fwd_workspace_size(const fhip_sdpa_paged_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_sdpa_paged_fwd_workspace_size: null");
  *bytes = 0;
  if (paged_validate(nullptr, d) != 0)
    return 1;
  if (fhip_fast_sdpa_paged_applicable(d))
    *bytes = fhip_fast_sdpa_paged_workspace(d);
  return 0;
}

int fhip_sdpa_paged_fwd_supported(const fhip_sdpa_paged_desc *d) {
  if (!d || paged_validate(nullptr, d) != 0)
    return 0;
  return fhip_fast_sdpa_paged_applicable(d) ? 2 : 1;
}

int fhip_sdpa_paged_fwd(fhip_ctx *ctx, const fhip_sdpa_paged_desc *d, const fhip_cache_ptrs *cache, const void *q,
                        const void *offsets, void *o, void *workspace, size_t workspace_bytes) {
  static const char who[] = "fhip_sdpa_paged_fwd";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (paged_validate(ctx, d) != 0 || fhip_check_cache_ptrs(ctx, who, d->cache, cache) != 0)
    return 1;
  FHIP_REQUIRE(ctx, q && offsets && o, "%s: null tensor pointer", who);
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  if (fhip_fast_sdpa_paged_applicable(d)) {
    if (check_workspace(ctx, who, fhip_fast_sdpa_paged_workspace(d), workspace, workspace_bytes))
      return 1;
    bool handled = false;
    const int rc = fhip_fast_sdpa_paged(ctx, d, cache, q, offsets, o, workspace, &handled);
    if (handled)
      return rc;
  }
  fhip_note_kernel(ctx, "sdpa_rows paged");
  RowsArgs g{};
  g.q = q, g.o = o, g.offsets = (const int32_t *)offsets;
  g.cache = fhip_cache_view(d->cache, *cache);
  g.batch = g.cache.batch, g.causal = d->is_causal != 0;
  return launch_rows(ctx, g, d->q, d->o, d->cache.k.dim[1], d->has_scale, d->scale);
}

} // extern "C"
