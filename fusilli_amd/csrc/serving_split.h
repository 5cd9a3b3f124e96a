// Which rows of packed tensors a sequence has, as kernels find it from device memory that no call has
// checked: plain arithmetic, the same on the host (tests/cpp/test_serving_split.cpp).
#ifndef FUSILLI_AMD_CSRC_SERVING_SPLIT_H
#define FUSILLI_AMD_CSRC_SERVING_SPLIT_H

#include <cstdint>

#if defined(__HIPCC__)
#define FHIP_SPLIT_FN __host__ __device__ __forceinline__
#else
#define FHIP_SPLIT_FN inline
#endif

// Rows begin .. end - 1 of T that offsets claim.  Both ends are clamped before the difference is taken, so that
// whatever they are neither it overflows nor first + count leaves 0 .. T.
struct FhipRows {
  int32_t first, count;
};
FHIP_SPLIT_FN FhipRows fhip_rows_between(int32_t begin, int32_t end, int32_t T) {
  const int32_t a = begin < 0 ? 0 : begin > T ? T : begin, e = end < 0 ? 0 : end > T ? T : end;
  return FhipRows{a, e > a ? e - a : 0};
}

#endif // FUSILLI_AMD_CSRC_SERVING_SPLIT_H
