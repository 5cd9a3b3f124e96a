// Rows to 8-bit codes with a scale each (fhip_quantize_rows), with an RMS norm or a swish gate
// in front.
#include "common.h"

#include <type_traits>

namespace {

struct QuantizeArgs {
  const void *x, *up, *weight;
  int8_t *q;
  float *scale;
  int64_t x_s[2], up_s[2], q_s[2], scale_s, weight_s;
  int64_t rows, K;
  int32_t dtype, weight_dt, front;
  float epsilon;
};

// A row's factors.  Below 2^-100 the factor 127 / a leaves f32's range, so both factors of
// y * (127 / a) are taken 2^64 times as large, which is exact.
struct RowScale {
  float scale, by, up; // code = rint(y * up * by)
};
__device__ __forceinline__ RowScale row_scale(float most, bool bad) {
  RowScale r;
  r.up = most < 0x1p-100f ? 0x1p64f : 1.f;
  r.scale = bad ? __builtin_nanf("") : most / 127.f;
  r.by = bad || most == 0.f ? 0.f : 127.f / (most * r.up);
  return r;
}
// As row_code, in the low byte of a word: adding 3 * 2^22 rounds to a whole number (ties to even, as
// rint), and no product is beyond 127 (1 + 2^-22).
__device__ __forceinline__ uint32_t held_code(float y, const RowScale &r) {
#pragma clang fp contract(off)
  return __builtin_bit_cast(uint32_t, y * r.up * r.by + 0x1.8p23f);
}
__device__ __forceinline__ int row_code(float y, const RowScale &r) {
  const float v = __builtin_rintf(y * r.up * r.by);
  return (int)fminf(fmaxf(v, -127.f), 127.f); // (NaN, of a row that is not finite: -127 * 0 below)
}

// x / (1 + exp(-x)) with the power of the negative one, e = exp(-|x|), which stays in range (it is 0
// from |x| = 104 on; an infinity or NaN in x stays one, or infinity times 0).  e is
// 2^t for t = -|x| log2(e), cut into its nearest whole number and a rest that is good to
// 2^-25: v_exp_f32 and v_rcp_f32 are good to a step each.  (The device library's exp and a whole
// division take three times the instructions, and this front is bound by them: see below.)
__device__ __forceinline__ float swish(float x) {
  const float a = fmaxf(-fabsf(x), -150.f), n = __builtin_rintf(a * 0x1.715476p+0f);
  const float rest = __builtin_fmaf(a, 0x1.4ae0cp-26f, __builtin_fmaf(a, 0x1.715476p+0f, -n));
  const float e = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(rest), (int)n);
  return (x < 0.f ? x * e : x) * __builtin_amdgcn_rcpf(1.f + e);
}

// 1 / sqrt(mean(x^2) + epsilon).  NaN where the squares' sum leaves f32, so that such a row counts as not finite.
__device__ __forceinline__ float norm_of(float sum, const QuantizeArgs &g) {
  return sum < INFINITY ? 1.f / sqrtf(sum / (float)g.K + g.epsilon) : __builtin_nanf("");
}

// y of one element (`norm`: 1 / sqrt(mean(x^2) + epsilon))
__device__ __forceinline__ float front_value(const QuantizeArgs &g, int64_t row, int64_t k, float norm) {
  float y = fhip_load<float>(g.x, g.dtype, row * g.x_s[0] + k * g.x_s[1]);
  if (g.front == FHIP_QUANTIZE_RMSNORM) {
    y *= norm;
    if (g.weight)
      y *= fhip_load<float>(g.weight, g.weight_dt, k * g.weight_s);
  } else if (g.front == FHIP_QUANTIZE_SWISH_GATE) {
    y = swish(y) * fhip_load<float>(g.up, g.dtype, row * g.up_s[0] + k * g.up_s[1]);
  }
  return y;
}

// Sums (or largest values) over a workgroup's wavefronts.
template <typename F> __device__ __forceinline__ float over_workgroup(float v, float *lds, F join) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1)
    v = join(v, __shfl_xor(v, d));
  const int waves = blockDim.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < waves; ++w)
    v = join(v, lds[w]);
  return v;
}

// Any strides and sizes: a workgroup a row, which is read again for each of the passes.
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs g) {
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    float norm = 1.f;
    if (g.front == FHIP_QUANTIZE_RMSNORM) {
      float sum = 0.f;
      for (int64_t k = threadIdx.x; k < g.K; k += 256) {
        const float x = fhip_load<float>(g.x, g.dtype, row * g.x_s[0] + k * g.x_s[1]);
        sum = __builtin_fmaf(x, x, sum);
      }
      sum = over_workgroup(sum, lds, [](float a, float b) { return a + b; });
      norm = norm_of(sum, g);
    }
    float most = 0.f, bad = 0.f;
    for (int64_t k = threadIdx.x; k < g.K; k += 256) {
      const float y = fabsf(front_value(g, row, k, norm));
      bad = y < INFINITY ? bad : 1.f;
      most = fmaxf(most, y);
    }
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    most = over_workgroup(most, lds, larger);
    bad = over_workgroup(bad, lds, larger);
    const RowScale r = row_scale(most, bad != 0.f);
    if (threadIdx.x == 0)
      g.scale[row * g.scale_s] = r.scale;
    for (int64_t k = threadIdx.x; k < g.K; k += 256)
      g.q[row * g.q_s[0] + k * g.q_s[1]] = bad != 0.f ? 0 : (int8_t)row_code(front_value(g, row, k, norm), r);
  }
}

// ---- rows with a last stride of 1, held in registers ------------------------------------------
//
// One pass over memory: each lane holds CHUNKS runs of 8 elements (16 or 32 bytes, loaded at the
// elements' alignment: a vector that starts inside a line costs one line more per wavefront), y in
// f32; the sum of squares and the largest |y| go over the lanes by DPP, over the wavefronts by LDS.
// |y| is compared by its bits, where infinities and NaN are the largest.
//
// Bound by memory where there are many rows: bf16 swish gate 4000 x 12288, 245 MB, 49.2 us (5.0 TB/s; the
// kernel of any strides below: 376 us), 16384 x 4096 without a front 38 us (5.3 TB/s); by the latency of a launch, a
// load and two reductions where there are few: 1 x 2048 with RMS norm 2.4 us, 48 x 8192 3.5 us.
typedef uint32_t QWord4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t QWord2 __attribute__((ext_vector_type(2), aligned(1)));
constexpr int kRun = 8;

// Eight elements as they are stored, and their values.
template <int DT> struct Run {
  static constexpr int N = DT == FHIP_FLOAT ? 2 : 1;
  uint32_t w[4 * N];
  __device__ __forceinline__ void load(const void *base, int64_t first, int live) {
    const char *p = (const char *)base + first * (DT == FHIP_FLOAT ? 4 : 2);
    if (live >= kRun) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const QWord4 v = ((const QWord4 *)p)[n];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[4 * n + i] = v[i];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4 * N; ++i)
      w[i] = 0;
    if (live <= 0)
      return;
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (i < live) {
        if constexpr (DT == FHIP_FLOAT)
          w[i] = ((const uint32_t *)p)[i];
        else
          w[i / 2] |= (uint32_t)((const uint16_t *)p)[i] << (16 * (i & 1));
      }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == FHIP_FLOAT)
      return __builtin_bit_cast(float, w[i]);
    else if constexpr (DT == FHIP_BFLOAT16)
      return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
};

// Over the 16 lanes of a DPP row; in each of them.
template <typename T, typename F> __device__ __forceinline__ T over_row(T v, F join) {
  auto step = [&](auto ctrl) {
    v = join(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF,
                                                                  0xF, false)));
  };
  step(std::integral_constant<int, 0xB1>{});  // quad_perm [1,0,3,2]
  step(std::integral_constant<int, 0x4E>{});  // quad_perm [2,3,0,1]
  step(std::integral_constant<int, 0x124>{}); // row_ror 4
  step(std::integral_constant<int, 0x128>{}); // row_ror 8
  return v;
}
// Over a row of `waves` wavefronts; 0 joined with v is v.  `lds`: 16 words that no other join uses.
template <bool ONE, typename T, typename F> __device__ __forceinline__ T over_waves(T v, uint32_t *lds, int waves, F join) {
  v = over_row(v, join);
  auto lane = [&](int l) { return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
  v = join(join(lane(0), lane(16)), join(lane(32), lane(48)));
  if constexpr (ONE)
    return v;
  if ((threadIdx.x & 63) == 0)
    lds[threadIdx.x >> 6] = __builtin_bit_cast(uint32_t, v);
  __syncthreads();
  const int at = threadIdx.x & 15;
  return over_row(at < waves ? __builtin_bit_cast(T, lds[at]) : T(0), join);
}

// ONE: rows of at most 512 elements, a wavefront each, four to a workgroup; otherwise a workgroup a row.
template <int DT, int FRONT, int CHUNKS, bool ONE>
__global__ __launch_bounds__(ONE ? 256 : 1024) void quantize_held_kernel(QuantizeArgs g) {
  __shared__ uint32_t lds[2][16];
  const int thread = ONE ? threadIdx.x & 63 : threadIdx.x, threads = ONE ? 64 : blockDim.x;
  const int64_t row = ONE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (ONE && row >= g.rows)
    return;
  const int K = (int)g.K;
  Run<DT> x[CHUNKS], up[CHUNKS];
  Run<FHIP_FLOAT> wide[CHUNKS]; // the weight: of X's type in its first half, or f32
  constexpr bool WEIGHT = FRONT == FHIP_QUANTIZE_RMSNORM;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int at = (c * threads + thread) * kRun;
    x[c].load(g.x, row * g.x_s[0] + at, K - at);
    if (FRONT == FHIP_QUANTIZE_SWISH_GATE)
      up[c].load(g.up, row * g.up_s[0] + at, K - at);
  }
  float y[CHUNKS][kRun];
  float norm = 1.f;
  if (WEIGHT) {
    if (g.weight) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int at = (c * threads + thread) * kRun;
        if (g.weight_dt == FHIP_FLOAT) {
          wide[c].load(g.weight, at, K - at);
        } else {
          Run<FHIP_BFLOAT16> w;
          w.load(g.weight, at, K - at);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            wide[c].w[i] = w.w[i];
        }
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        sum = __builtin_fmaf(x[c][i], x[c][i], sum);
    norm = norm_of(over_waves<ONE>(sum, lds[0], threads >> 6, [](float a, float b) { return a + b; }), g);
  }
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      y[c][i] = x[c][i];
      if (WEIGHT)
        y[c][i] *= norm;
      if (FRONT == FHIP_QUANTIZE_SWISH_GATE)
        y[c][i] = swish(y[c][i]) * up[c][i];
    }
    if (WEIGHT && g.weight) {
      auto times = [&](auto w) {
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          y[c][i] *= w(i);
      };
      if (g.weight_dt == FHIP_FLOAT) {
        times([&](int i) { return wide[c][i]; });
      } else if (g.weight_dt == FHIP_BFLOAT16) {
        times([&](int i) { return ((const Run<FHIP_BFLOAT16> &)wide[c])[i]; });
      } else {
        times([&](int i) { return ((const Run<FHIP_HALF> &)wide[c])[i]; });
      }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const uint32_t size = __builtin_bit_cast(uint32_t, y[c][i]) & 0x7FFFFFFFu;
      most = size > most ? size : most;
    }
  }
  most = over_waves<ONE>(most, lds[1], threads >> 6, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const bool bad = most >= 0x7F800000u;
  const RowScale r = row_scale(__builtin_bit_cast(float, most), bad);
  if (thread == 0)
    g.scale[row * g.scale_s] = r.scale;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int at = (c * threads + thread) * kRun, live = K - at;
    int8_t *q = g.q + row * g.q_s[0] + at;
    uint32_t code[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      code[i] = bad ? 0u : held_code(y[c][i], r);
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) // the low bytes of four codes
      out[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(code[4 * h + 3], code[4 * h + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(code[4 * h + 1], code[4 * h], 0x0C0C0400u), 0x05040100u);
    if (live >= kRun) {
      *(QWord2 *)q = QWord2{out[0], out[1]};
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (i < live)
          q[i] = (int8_t)(out[i / 4] >> (8 * (i & 3)));
    }
  }
}

// How the register kernel takes a row: the fewest runs per lane that 1024 threads allow.  bf16, 1 / 2 / 4
// runs: 1 x 2048 with RMS norm 2.4 / 2.8 / 3.5 us, 48 x 4096 2.8 / 3.2 / 3.9, 4096 x 4096
// 16.1 / 15.6 / 17.5, 16384 x 4096 alone 38.0 / 36.2 / 36.9.
struct Held {
  int chunks, threads;
  bool one;
  explicit Held(int64_t K) {
    const int runs = (int)((K + kRun - 1) / kRun);
    one = runs <= 64;
    chunks = runs <= 1024 ? 1 : runs <= 2048 ? 2 : 4;
    threads = one ? 256 : (((runs + chunks - 1) / chunks + 63) & ~63);
  }
};

template <int DT, int FRONT> void launch_held(fhip_ctx *ctx, const QuantizeArgs &g) {
  const Held h(g.K);
  const dim3 grid((unsigned)(h.one ? (g.rows + 3) / 4 : g.rows)), block(h.threads);
  if (h.one)
    hipLaunchKernelGGL((quantize_held_kernel<DT, FRONT, 1, true>), grid, block, 0, ctx->stream, g);
  else if (h.chunks == 1)
    hipLaunchKernelGGL((quantize_held_kernel<DT, FRONT, 1, false>), grid, block, 0, ctx->stream, g);
  else if (h.chunks == 2)
    hipLaunchKernelGGL((quantize_held_kernel<DT, FRONT, 2, false>), grid, block, 0, ctx->stream, g);
  else
    hipLaunchKernelGGL((quantize_held_kernel<DT, FRONT, 4, false>), grid, block, 0, ctx->stream, g);
}
template <int DT> void launch_held(fhip_ctx *ctx, const QuantizeArgs &g) {
  if (g.front == FHIP_QUANTIZE_RMSNORM)
    launch_held<DT, FHIP_QUANTIZE_RMSNORM>(ctx, g);
  else if (g.front == FHIP_QUANTIZE_SWISH_GATE)
    launch_held<DT, FHIP_QUANTIZE_SWISH_GATE>(ctx, g);
  else
    launch_held<DT, FHIP_QUANTIZE_NONE>(ctx, g);
}

constexpr int64_t kHeldK = 4 * 1024 * kRun;
// (a grid has fewer than 2^32 threads)
bool held(const fhip_quantize_rows_desc &d) {
  auto dense = [](const fhip_tensor_desc &t) { return t.dim[1] == 1 || t.stride[1] == 1; };
  return d.x.dim[1] <= kHeldK && d.x.dim[0] < (1 << 21) && dense(d.x) && dense(d.q) && (!d.up.rank || dense(d.up)) &&
         (!d.has_weight || d.weight_stride == 1 || d.x.dim[1] == 1);
}

bool is_float(int dt) { return dt == FHIP_FLOAT || dt == FHIP_BFLOAT16 || dt == FHIP_HALF; }

} // namespace

static int validate(fhip_ctx *ctx, const fhip_quantize_rows_desc *d) {
  static const char who[] = "fhip_quantize_rows";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (!fhip_check_desc(ctx, d->x, "quantize X") || !fhip_check_desc(ctx, d->q, "quantize Q"))
    return 1;
  FHIP_REQUIRE(ctx, d->x.rank == 2 && d->q.rank == 2 && d->x.dim[0] == d->q.dim[0] && d->x.dim[1] == d->q.dim[1],
               "%s: X and Q must be [rows, K]", who);
  FHIP_REQUIRE(ctx, is_float(d->x.dtype), "%s: X must be f32, bf16 or f16", who);
  FHIP_REQUIRE(ctx, d->q.dtype == FHIP_INT8, "%s: Q must be Int8", who);
  FHIP_REQUIRE(ctx, (d->q.dim[0] == 1 || d->q.stride[0] > 0) && (d->q.dim[1] == 1 || d->q.stride[1] > 0),
               "%s: Q has a stride of 0", who);
  FHIP_REQUIRE(ctx, d->scale_stride > 0 || (d->scale_stride == 0 && d->x.dim[0] == 1), "%s: scale_stride must be above 0",
               who);
  FHIP_REQUIRE(ctx, d->front >= FHIP_QUANTIZE_NONE && d->front <= FHIP_QUANTIZE_SWISH_GATE, "%s: unknown front %d", who,
               d->front);
  FHIP_REQUIRE(ctx, (d->up.rank != 0) == (d->front == FHIP_QUANTIZE_SWISH_GATE), "%s: UP and the swish gate go together",
               who);
  if (d->up.rank) {
    if (!fhip_check_desc(ctx, d->up, "quantize UP"))
      return 1;
    FHIP_REQUIRE(ctx, d->up.rank == 2 && d->up.dim[0] == d->x.dim[0] && d->up.dim[1] == d->x.dim[1] &&
                          d->up.dtype == d->x.dtype,
                 "%s: UP must have X's dims and type", who);
  }
  FHIP_REQUIRE(ctx, !d->has_weight || d->front == FHIP_QUANTIZE_RMSNORM, "%s: a weight needs the RMS norm", who);
  FHIP_REQUIRE(ctx, !d->has_weight || (is_float(d->weight_dtype) && d->weight_stride >= 0),
               "%s: the weight must be f32, bf16 or f16 with a stride that is not negative", who);
  FHIP_REQUIRE(ctx, d->front != FHIP_QUANTIZE_RMSNORM || d->epsilon >= 0.f, "%s: epsilon must not be negative", who);
  return 0;
}

extern "C" {

int fhip_quantize_rows_workspace_size(const fhip_quantize_rows_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_quantize_rows_workspace_size: null");
  *bytes = 0;
  return 0;
}

int fhip_quantize_rows_supported(const fhip_quantize_rows_desc *d) {
  if (!d || validate(nullptr, d) != 0)
    return 0;
  return held(*d) ? 2 : 1;
}

int fhip_quantize_rows(fhip_ctx *ctx, const fhip_quantize_rows_desc *d, const void *x, const void *up, const void *weight,
                       void *q, void *scale, void *workspace, size_t workspace_bytes) {
  static const char who[] = "fhip_quantize_rows";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (validate(ctx, d) != 0)
    return 1;
  FHIP_REQUIRE(ctx, x && q && scale, "%s: null tensor pointer", who);
  FHIP_REQUIRE(ctx, (d->up.rank != 0) == (up != nullptr), "%s: UP pointer and descriptor disagree", who);
  FHIP_REQUIRE(ctx, (d->has_weight != 0) == (weight != nullptr), "%s: weight and has_weight disagree", who);
  (void)workspace;
  (void)workspace_bytes;
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  QuantizeArgs g{};
  g.x = x, g.up = up, g.weight = weight, g.q = (int8_t *)q, g.scale = (float *)scale;
  for (int i = 0; i < 2; ++i)
    g.x_s[i] = d->x.stride[i], g.up_s[i] = d->up.stride[i], g.q_s[i] = d->q.stride[i];
  g.scale_s = d->scale_stride, g.weight_s = d->weight_stride;
  g.rows = d->x.dim[0], g.K = d->x.dim[1];
  g.dtype = d->x.dtype, g.weight_dt = d->weight_dtype, g.front = d->front, g.epsilon = d->epsilon;
  if (held(*d)) {
    fhip_note_kernel(ctx, "quantize_rows_held");
    if (g.dtype == FHIP_FLOAT)
      launch_held<FHIP_FLOAT>(ctx, g);
    else if (g.dtype == FHIP_BFLOAT16)
      launch_held<FHIP_BFLOAT16>(ctx, g);
    else
      launch_held<FHIP_HALF>(ctx, g);
    FHIP_HIP_CHECK(ctx, hipGetLastError());
    return 0;
  }
  fhip_note_kernel(ctx, "quantize_rows_generic");
  const int64_t most = (int64_t)ctx->num_cus * 32;
  hipLaunchKernelGGL(quantize_rows_kernel, dim3((unsigned)(g.rows < most ? g.rows : most)), dim3(256), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
