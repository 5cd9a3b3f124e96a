// Packed sequences and a key / value cache in pages, as kernels see them: which
// sequence a row belongs to, where a key lies, and what 4-bit codes stand for.
// Offsets, lengths and page numbers come from device memory that no call has
// checked: every lookup here stays inside the tensors whatever they hold.
#ifndef FUSILLI_AMD_CSRC_PAGED_CACHE_H
#define FUSILLI_AMD_CSRC_PAGED_CACHE_H

#include "common.h"
#include "serving_split.h"

constexpr int kCacheMaxDim = 512; // of a head
// Scales that the tuned attention kernels take: their maxima are those of raw scores and begin at -1e30, whose multiple by
// the scale has to stay a number (above, a row that sees nothing of a chunk would be exp2(-inf + inf)).
constexpr float kCacheMaxScale = 1e8f;
inline bool fhip_tuned_scale(bool has_scale, float scale) {
  return !has_scale || (scale > 0.f && scale <= kCacheMaxScale);
}
constexpr int64_t kCacheMaxKeys = (1ll << 30); // of a sequence: places stay 32-bit numbers

// One pool of a cache: K or V.  Strides in elements (bytes, in 4 bits).
struct FhipPool {
  char *data;
  _Float16 *params; // null: not in 4 bits
  int64_t page, head, slot;                   // strides of data
  int64_t params_page, params_head, params_slot;
};

struct FhipCacheView {
  FhipPool k, v;
  const int32_t *table, *lengths;
  int64_t table_stride;
  int32_t batch, table_pages; // rows and columns of the table
  int32_t pool_pages, page_size;
  int32_t group;              // elements per (scale, low) pair; 0: the pool's own type
  int32_t dtype;              // of the pools, without 4 bits
};

FhipCacheView fhip_cache_view(const fhip_cache_desc &c, const fhip_cache_ptrs &p);

// The checks that append, read and attention share: a cache of `heads` heads of K rows
// of `D` and V rows of `Dv` elements of type `dtype` (or 4 bits).
int fhip_check_cache(fhip_ctx *ctx, const char *who, const fhip_cache_desc &c, int dtype,
                     int64_t heads, int64_t D, int64_t Dv);
int fhip_check_cache_ptrs(fhip_ctx *ctx, const char *who, const fhip_cache_desc &c,
                          const fhip_cache_ptrs *p);
// A rank-3 tensor [rows, heads, dim] of f32, bf16 or f16 with neighbouring elements side
// by side.  `written`: no two elements may share memory, as far as strides of 0 say.
int fhip_check_rows(fhip_ctx *ctx, const char *who, const char *what, const fhip_tensor_desc &t,
                    bool written);

#if defined(__HIPCC__)

// Sequence of packed row `row`: the last b with offsets[b] <= row, so that rows of empty
// sequences are skipped; -1 where the row lies in front of the first or behind the last.
__device__ __forceinline__ int fhip_sequence_of(const int32_t *offsets, int batch, int row) {
  int lo = 0, hi = batch; // offsets[lo] <= row < offsets[hi]
  if (row < offsets[0] || row >= offsets[batch])
    return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Page of key `j` of sequence `b`, -1 where the table or the pool has none.
__device__ __forceinline__ int fhip_page_of(const FhipCacheView &c, int b, int j) {
  const uint32_t i = (uint32_t)j / (uint32_t)c.page_size;
  if (j < 0 || i >= (uint32_t)c.table_pages)
    return -1;
  const int page = c.table[b * c.table_stride + i];
  return (uint32_t)page < (uint32_t)c.pool_pages ? page : -1;
}

// Element e of the row at (page, slot) of head h as a float.
__device__ __forceinline__ float fhip_cache_value(const FhipCacheView &c, const FhipPool &p, int page, int slot,
                                                  int h, int e) {
  const int64_t at = page * p.page + h * p.head + slot * p.slot;
  if (!c.group)
    return fhip_load<float>(p.data, c.dtype, at + e);
  const uint8_t two = ((const uint8_t *)p.data)[at + e / 2];
  const _Float16 *pair = p.params + page * p.params_page + h * p.params_head + slot * p.params_slot + e / c.group * 2;
  return (float)pair[1] + (float)pair[0] * (float)(e & 1 ? two >> 4 : two & 15);
}

// (scale, low) of a group of values from `lo` to `hi`, both NaN where `lo` or `hi` is no
// number or half cannot hold them.  Every step is a single rounding in f32 (no fused
// multiply-add), so that the same formula anywhere gives the same codes.
struct FhipGroup {
  _Float16 scale, low;
  float by; // 1 / scale, 0 where the codes are 0
};
__device__ __forceinline__ FhipGroup fhip_group_of(float lo, float hi) {
#pragma clang fp contract(off)
  FhipGroup g;
  g.low = (_Float16)lo;
  const float l = (float)g.low;
  float wide = hi - l;
  wide = wide < 0.f ? 0.f : wide;
  // wide / 15, correctly rounded: the quotient by the rounded reciprocal is within a step, and the exact remainder
  // times the reciprocal takes it the rest of the way (infinite: NaN, refused below like infinity)
  const float q = wide * (1.0f / 15.0f);
  float part = __builtin_fmaf(__builtin_fmaf(-15.0f, q, wide), 1.0f / 15.0f, q);
  asm("" : "+v"(part)); // (or the compiler rounds the sum to half at once)
  g.scale = (_Float16)part;
  const float s = (float)g.scale;
  if (!(__builtin_fabsf(l) < INFINITY) || !(s < INFINITY)) {
    g.scale = g.low = (_Float16)__builtin_nanf("");
    g.by = 0.f;
  } else {
    // 1 / s, correctly rounded: one step from the hardware's reciprocal, a unit off at most, leaves 2^-46, and the
    // reciprocal of an 11-bit number lies 2^-36 or more from where rounding changes (or is a power of two, exact)
    const float r = __builtin_amdgcn_rcpf(s);
    g.by = s > 0.f ? __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r) : 0.f;
  }
  return g;
}
// The code of x as a float, 0 for a NaN.
__device__ __forceinline__ float fhip_code_of(const FhipGroup &g, float x) {
#pragma clang fp contract(off)
  return __builtin_rintf(fminf(fmaxf((x - (float)g.low) * g.by, 0.f), 15.f));
}
// 8 codes of a word, the first in its lowest bits.  Added to 1.5 * 2^23 a number below 2^22 is rounded to an
// integer, half to even, which lies in the sum's lowest bits; the rest is the same in every sum and comes off at the end.
__device__ __forceinline__ uint32_t fhip_codes_of(const FhipGroup &g, const float (&x)[8]) {
#pragma clang fp contract(off)
  uint32_t w = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float c = fminf(fmaxf((x[i] - (float)g.low) * g.by, 0.f), 15.f) + 12582912.0f;
    w = (w << 4) + __builtin_bit_cast(uint32_t, c);
  }
  return w - 0x4b400000u * 0x11111111u;
}

#endif // __HIPCC__

#endif // FUSILLI_AMD_CSRC_PAGED_CACHE_H
