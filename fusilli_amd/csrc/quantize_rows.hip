// Rows to 8-bit codes with a scale each (fhip_quantize_rows), with an RMS norm or a swish gate
// in front.
#include "common.h"

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
__device__ __forceinline__ int row_code(float y, const RowScale &r) {
  const float v = __builtin_rintf(y * r.up * r.by);
  return (int)fminf(fmaxf(v, -127.f), 127.f); // (NaN, of a row that is not finite: -127 * 0 below)
}

// y of one element (`norm`: 1 / sqrt(mean(x^2) + epsilon))
__device__ __forceinline__ float front_value(const QuantizeArgs &g, int64_t row, int64_t k, float norm) {
  float y = fhip_load<float>(g.x, g.dtype, row * g.x_s[0] + k * g.x_s[1]);
  if (g.front == FHIP_QUANTIZE_RMSNORM) {
    y *= norm;
    if (g.weight)
      y *= fhip_load<float>(g.weight, g.weight_dt, k * g.weight_s);
  } else if (g.front == FHIP_QUANTIZE_SWISH_GATE) {
    y = y / (1.f + expf(-y)) * fhip_load<float>(g.up, g.dtype, row * g.up_s[0] + k * g.up_s[1]);
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
      norm = 1.f / sqrtf(sum / (float)g.K + g.epsilon);
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
  return 1;
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
  fhip_note_kernel(ctx, "quantize_rows_generic");
  const int64_t most = (int64_t)ctx->num_cus * 32;
  hipLaunchKernelGGL(quantize_rows_kernel, dim3((unsigned)(g.rows < most ? g.rows : most)), dim3(256), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
