// Product of 8-bit codes with scales per row and column (fhip_matmul_quantized): validation, the
// choice of kernels and the one for any strides.
//
// C = fma(sum * a_scale, b_scale, bias) with a whole sum: codes are -128 at the lowest, and 2^14 K is below 2^31 up to
// K = 131071.  The sums are scaled where the three families of products finish their tiles, so
// that a split of K adds whole numbers and changes no result.  Bound by the matrix pipes from a few hundred rows on
// (4096 x 8192 x 4096 into bf16 106-113 us, 2.4 to 2.6 POP/s), by the weights below (5 x 4096 x 131072 into
// f32 90 us, 5.9 TB/s; 48 x 4096 x 12288 12.9, 3.9 TB/s), by a launch, the first loads and the epilogue for small ones
// (1 x 2048 x 2560 4.6).
#include "fast_paths.h"

namespace {

struct ScaledArgs {
  const int8_t *a, *b;
  void *out;
  FhipProductScales scales;
  int64_t a_s[2], b_s[2], o_s[2];
  int64_t M, N, K;
  int32_t c_dt, o_dt;
  DevEpilogue epi;
};

// Any strides: a thread per result.
__global__ __launch_bounds__(256) void matmul_quantized_kernel(ScaledArgs g) {
  const int64_t total = g.M * g.N, step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += step) {
    const int64_t m = at / g.N, n = at - m * g.N;
    const int8_t *a = g.a + m * g.a_s[0], *b = g.b + n * g.b_s[1];
    int sum = 0;
    for (int64_t k = 0; k < g.K; ++k)
      sum += (int)a[k * g.a_s[1]] * (int)b[k * g.b_s[0]];
    float v = fhip_scaled(sum, g.scales.row(m), g.scales.column(n), g.scales.bias_of(n));
    v = fhip_round_through<float>(g.c_dt, v);
    const int64_t coord[2] = {m, n};
    v = fhip_apply_epilogue<float>(g.epi, v, coord);
    fhip_store<float>(g.out, g.o_dt, m * g.o_s[0] + n * g.o_s[1], v);
  }
}

bool is_float(int dt) { return dt == FHIP_FLOAT || dt == FHIP_BFLOAT16 || dt == FHIP_HALF; }

} // namespace

// The product as fhip_matmul's kernels have it.
static fhip_matmul_desc matmul_of(const fhip_matmul_quantized_desc &d) {
  fhip_matmul_desc m;
  m.a = d.a, m.b = d.b, m.c = d.c, m.out = d.out;
  m.epilogue = d.epilogue;
  m.out_dtype = d.out_dtype;
  return m;
}

static int validate(fhip_ctx *ctx, const fhip_matmul_quantized_desc *d) {
  static const char who[] = "fhip_matmul_quantized";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (!fhip_check_desc(ctx, d->a, "quantized matmul A") || !fhip_check_desc(ctx, d->b, "quantized matmul B") ||
      !fhip_check_desc(ctx, d->c, "quantized matmul C") || !fhip_check_desc(ctx, d->out, "quantized matmul OUT"))
    return 1;
  FHIP_REQUIRE(ctx, d->a.rank == 2 && d->b.rank == 2 && d->c.rank == 2 && d->out.rank == 2,
               "%s: A, B, C and OUT must be matrices", who);
  FHIP_REQUIRE(ctx, d->a.dtype == FHIP_INT8 && d->b.dtype == FHIP_INT8, "%s: A and B must be Int8", who);
  FHIP_REQUIRE(ctx, d->a.dim[1] == d->b.dim[0], "%s: K mismatch (%lld vs %lld)", who, (long long)d->a.dim[1],
               (long long)d->b.dim[0]);
  // (131071 products of -128 and -128 are 2^31 - 2^14)
  FHIP_REQUIRE(ctx, d->a.dim[1] <= 131071, "%s: K = %lld is above 131071, where sums may leave 32 bits", who,
               (long long)d->a.dim[1]);
  FHIP_REQUIRE(ctx, d->c.dim[0] == d->a.dim[0] && d->c.dim[1] == d->b.dim[1], "%s: C dims do not match M x N", who);
  FHIP_REQUIRE(ctx, d->out.dim[0] == d->c.dim[0] && d->out.dim[1] == d->c.dim[1], "%s: OUT dims differ from C dims", who);
  FHIP_REQUIRE(ctx, is_float(d->c.dtype), "%s: C must be f32, bf16 or f16", who);
  FHIP_REQUIRE(ctx, d->out.dtype == d->out_dtype, "%s: out_dtype disagrees with OUT descriptor", who);
  for (int i = 0; i < 2; ++i)
    FHIP_REQUIRE(ctx, d->out.dim[i] == 1 || d->out.stride[i] > 0, "%s: OUT has a stride of 0", who);
  FHIP_REQUIRE(ctx, d->a_scale_stride >= 0 && d->b_scale_stride >= 0, "%s: negative stride between scales", who);
  FHIP_REQUIRE(ctx, !d->has_bias || (is_float(d->bias_dtype) && d->bias_stride >= 0),
               "%s: the bias must be f32, bf16 or f16 with a stride that is not negative", who);
  return 0;
}

extern "C" {

int fhip_matmul_quantized_workspace_size(const fhip_matmul_quantized_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_matmul_quantized_workspace_size: null");
  *bytes = 0;
  return 0;
}

int fhip_matmul_quantized_supported(const fhip_matmul_quantized_desc *d) {
  if (!d || validate(nullptr, d) != 0)
    return 0;
  const fhip_matmul_desc m = matmul_of(*d);
  return fhip_fast_matmul_applicable(&m, true) ? 2 : 1;
}

int fhip_matmul_quantized(fhip_ctx *ctx, const fhip_matmul_quantized_desc *d, const void *a, const void *b,
                          const void *a_scale, const void *b_scale, const void *bias, const void *const *epilogue_operands,
                          void *out, void *workspace, size_t workspace_bytes) {
  static const char who[] = "fhip_matmul_quantized";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (validate(ctx, d) != 0)
    return 1;
  FHIP_REQUIRE(ctx, a && b && a_scale && b_scale && out, "%s: null tensor pointer", who);
  FHIP_REQUIRE(ctx, (d->has_bias != 0) == (bias != nullptr), "%s: bias and has_bias disagree", who);
  (void)workspace;
  (void)workspace_bytes;
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  DevEpilogue epi;
  if (fhip_build_epilogue(ctx, d->epilogue, 2, d->c.dim, epilogue_operands, &epi) != 0)
    return 1;
  FhipProductScales s{};
  s.a = (const float *)a_scale, s.b = (const float *)b_scale, s.bias = bias;
  s.a_s = d->a_scale_stride, s.b_s = d->b_scale_stride, s.bias_s = d->bias_stride, s.bias_dt = d->bias_dtype;
  const fhip_matmul_desc md = matmul_of(*d);
  bool handled = false, short_k = false;
  const int rc = fhip_tuned_matmul(ctx, &md, a, b, epi, out, &handled, &short_k, &s);
  if (handled)
    return rc;
  fhip_note_kernel(ctx, "matmul_quantized_generic");
  ScaledArgs g{};
  g.a = (const int8_t *)a, g.b = (const int8_t *)b, g.out = out, g.scales = s;
  for (int i = 0; i < 2; ++i)
    g.a_s[i] = d->a.stride[i], g.b_s[i] = d->b.stride[i], g.o_s[i] = d->out.stride[i];
  g.M = d->a.dim[0], g.N = d->b.dim[1], g.K = d->a.dim[1];
  g.c_dt = d->c.dtype, g.o_dt = d->out.dtype, g.epi = epi;
  const int64_t blocks = (g.M * g.N + 255) / 256, most = (int64_t)ctx->num_cus * 32;
  hipLaunchKernelGGL(matmul_quantized_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
