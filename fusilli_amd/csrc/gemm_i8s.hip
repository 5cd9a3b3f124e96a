// MFMA GEMM kernels for i8 operands whose sums are scaled by row and column.
#include "gemm_kernel.h"

int gemm_launch_i8s(fhip_ctx *ctx, const GemmPlan &p, const GemmArgs &g) {
  return gemm_launch_kind<GK_I8S>(ctx, p, g);
}
