// Direct matrix-product kernels for i8 operands whose sums are scaled.
#include "gemm_direct_kernel.h"

int direct_launch_i8s(fhip_ctx *ctx, const DirectPlan &p, const DirectArgs &g, int64_t batch) {
  return direct_launch_kind<GK_I8S>(ctx, p, g, batch);
}
