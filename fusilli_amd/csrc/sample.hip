// A token for each row of logits from given random numbers (fhip_sample).
//
// Words are ordered by their logits, the largest first, equal ones by their index.  What
// temperature, top-k, top-p and min-p keep is the first so many in that order, and the token is the
// first up to which the kept weights' sum exceeds uniform times all of it; so every question is for
// a prefix of the order: up to a count, up to a sum.  None of them needs the words sorted: a
// prefix ends in one value of the logits, found digit by digit from counts and sums of the words
// that share the digits above, and in one of the words that have that value, by index.
//
// Weights exp((l - m) / T) are f64 and kept as whole multiples of 2^-40, so that sums are exact
// in 64 bits whatever the order of the additions (2^24 words stay below 2^64): the same token on
// every run and from every way of cutting the row.  A weight's rounding is 2^-41 of the
// largest, 2^17 times less than f32 would leave.
#include "common.h"

namespace {

struct SampleArgs {
  const void *logits;
  const float *uniform, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int32_t *token;
  float *probability;
  int64_t row_s, word_s;
  int64_t rows;
  int32_t words, dtype;
  float one_temperature, one_top_p, one_min_p;
  int32_t one_top_k;
};

constexpr double kUnit = 1099511627776.0; // 2^40

// Ascending with the logit: 0 for what is never drawn (NaN, -inf); -0 is 0.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -INFINITY))
    return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Settings {
  double most, by; // the largest logit; 1 / T as a divisor: T
  bool greedy;
  __device__ __forceinline__ double weight(uint32_t key) const { // of a word that may be drawn
    const double l = (double)logit_of(key);
    return l == most ? 1.0 : exp((l - most) / by);
  }
  __device__ __forceinline__ uint64_t held(uint32_t key) const { return (uint64_t)rint(weight(key) * kUnit); }
};

// The end of a prefix: the last value that it holds, how many words have larger ones and their
// weights, and how many words of that value it takes.
struct End {
  uint32_t key;
  uint32_t count;
  uint64_t sum;
  uint32_t ties;
};

constexpr int kThreads = 256;

struct Shared {
  uint64_t sum[256];
  uint32_t count[256];
  uint32_t digit;
  uint32_t above_count;
  uint64_t above_sum;
  uint64_t wave[kThreads / 64];
};

template <typename F> __device__ __forceinline__ uint64_t over_workgroup(uint64_t v, Shared &s, F join) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1)
    v = join(v, (uint64_t)__shfl_xor((unsigned long long)v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    s.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.wave[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w)
    v = join(v, s.wave[w]);
  return v;
}

// The end of the shortest prefix that holds `need` words (by_count) or whose weights' sum is at
// least `need`; the row has as much.
template <typename Key>
__device__ __forceinline__ End find_end(bool by_count, uint64_t need, int words, const Settings &set, Shared &s, Key key_at) {
  uint32_t prefix = 0;
  uint32_t count = 0;
  uint64_t sum = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads)
      s.sum[i] = 0, s.count[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < words; i += kThreads) {
      const uint32_t key = key_at(i);
      if (key == 0 || (shift < 24 && key >> (shift + 8) != prefix))
        continue;
      const int digit = (int)(key >> shift & 255);
      atomicAdd(&s.count[digit], 1u);
      atomicAdd((unsigned long long *)&s.sum[digit], (unsigned long long)set.held(key));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t c = count;
      uint64_t w = sum;
      int digit = 255, last = -1;
      for (; digit >= 0; --digit) {
        if (s.count[digit] == 0)
          continue;
        last = digit;
        if (by_count ? c + s.count[digit] >= need : w + s.sum[digit] >= need)
          break;
        c += s.count[digit], w += s.sum[digit];
      }
      if (digit < 0) { // (never, as the row has as much)
        digit = last < 0 ? 0 : last;
        c -= s.count[digit], w -= s.sum[digit];
      }
      s.digit = (uint32_t)digit, s.above_count = c, s.above_sum = w;
    }
    __syncthreads();
    prefix = prefix << 8 | s.digit;
    count = s.above_count, sum = s.above_sum;
  }
  End e;
  e.key = prefix, e.count = count, e.sum = sum;
  const uint32_t same = s.count[s.digit];
  const uint64_t each = set.held(prefix);
  uint64_t ties = by_count ? need - count : need <= sum ? 1 : each == 0 ? 1 : (need - sum + each - 1) / each;
  e.ties = (uint32_t)(ties < 1 ? 1 : ties > same ? same : ties);
  __syncthreads();
  return e;
}

// Any strides and sizes: a workgroup a row, which is read again for each digit.
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(SampleArgs g) {
  __shared__ Shared s;
  __shared__ int found;
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    auto key_at = [&](int i) { return key_of(fhip_load<float>(g.logits, g.dtype, row * g.row_s + i * g.word_s)); };
    uint64_t most = 0, some = 0;
    for (int i = threadIdx.x; i < g.words; i += kThreads) {
      const uint32_t key = key_at(i);
      most = key > most ? key : most;
      some += key != 0;
    }
    most = over_workgroup(most, s, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    some = over_workgroup(some, s, [](uint64_t a, uint64_t b) { return a + b; });
    if (some == 0) {
      if (threadIdx.x == 0) {
        g.token[row] = -1;
        if (g.probability)
          g.probability[row] = 0.f;
      }
      continue;
    }
    const float t = g.temperature ? g.temperature[row] : g.one_temperature;
    const int k = g.top_k ? g.top_k[row] : g.one_top_k;
    const float p = g.top_p ? g.top_p[row] : g.one_top_p, least = g.min_p ? g.min_p[row] : g.one_min_p;
    const float u = g.uniform[row];
    Settings set;
    set.most = (double)logit_of((uint32_t)most);
    set.greedy = !(t > 0.f);
    set.by = set.greedy ? 1.0 : (double)t;
    uint64_t kept = (uint64_t)kUnit; // (greedy: the first word's weight)
    if (!set.greedy) {
      // what the first k weigh
      if (k > 0 && (uint64_t)k < some) {
        const End e = find_end(true, (uint64_t)k, g.words, set, s, key_at);
        kept = e.sum + e.ties * set.held(e.key);
      } else {
        kept = 0;
        for (int i = threadIdx.x; i < g.words; i += kThreads)
          if (const uint32_t key = key_at(i))
            kept += set.held(key);
        kept = over_workgroup(kept, s, [](uint64_t a, uint64_t b) { return a + b; });
      }
      uint64_t strict = kept;
      if (p < 1.f) {
        const double share = p > 0.f ? ceil((double)p * (double)kept) : 1.0;
        const uint64_t need = share < (double)kept ? (uint64_t)share : kept;
        const End e = find_end(false, need < 1 ? 1 : need, g.words, set, s, key_at);
        strict = e.sum + e.ties * set.held(e.key);
      }
      if (least > 0.f) {
        uint64_t large = 0;
        const double bound = least < 1.f ? (double)least : 1.0;
        for (int i = threadIdx.x; i < g.words; i += kThreads) {
          const uint32_t key = key_at(i);
          if (key && set.weight(key) >= bound)
            large += set.held(key);
        }
        large = over_workgroup(large, s, [](uint64_t a, uint64_t b) { return a + b; });
        strict = large < strict ? large : strict;
      }
      kept = strict < kept ? strict : kept;
      if (least > 1.f)
        kept = (uint64_t)kUnit;
    }
    // the first word up to which the sum is above u * kept
    const double at = set.greedy || !(u > 0.f) ? 0.0 : floor((double)u * (double)kept);
    const uint64_t above = at < (double)kept ? (uint64_t)at : kept - 1;
    const End e = find_end(false, (above < kept ? above : kept - 1) + 1, g.words, set, s, key_at);
    // its index: the `ties`-th of its value
    if (threadIdx.x == 0)
      found = -1;
    uint32_t left = e.ties;
    for (int from = 0; from < g.words; from += kThreads) {
      const int i = from + threadIdx.x;
      const bool here = i < g.words && key_at(i) == e.key;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(here);
      __syncthreads();
      if ((threadIdx.x & 63) == 0)
        s.wave[threadIdx.x >> 6] = (uint64_t)__builtin_popcountll(mask);
      __syncthreads();
      uint32_t before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) {
        before += w < (int)(threadIdx.x >> 6) ? (uint32_t)s.wave[w] : 0u;
        all += (uint32_t)s.wave[w];
      }
      if (left > all) {
        left -= all;
        continue;
      }
      before += (uint32_t)__builtin_popcountll(mask & ((1ull << (threadIdx.x & 63)) - 1));
      if (here && before + 1 == left)
        found = i;
      break; // (uniform: `left` and `all` are)
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      g.token[row] = found;
      if (g.probability)
        g.probability[row] = (float)((double)set.held(e.key) / (double)kept);
    }
    __syncthreads();
  }
}

bool is_float(int dt) { return dt == FHIP_FLOAT || dt == FHIP_BFLOAT16 || dt == FHIP_HALF; }

} // namespace

static int validate(fhip_ctx *ctx, const fhip_sample_desc *d) {
  static const char who[] = "fhip_sample";
  FHIP_REQUIRE(ctx, d != nullptr, "%s: null descriptor", who);
  if (!fhip_check_desc(ctx, d->logits, "sample LOGITS"))
    return 1;
  FHIP_REQUIRE(ctx, d->logits.rank == 2, "%s: LOGITS must be [rows, words]", who);
  FHIP_REQUIRE(ctx, is_float(d->logits.dtype), "%s: LOGITS must be f32, bf16 or f16", who);
  FHIP_REQUIRE(ctx, d->logits.dim[1] <= (1 << 24), "%s: more than 2^24 words", who);
  FHIP_REQUIRE(ctx, d->logits.dim[0] < (1ll << 31), "%s: more than 2^31 - 1 rows", who);
  return 0;
}

extern "C" {

int fhip_sample_workspace_size(const fhip_sample_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_sample_workspace_size: null");
  *bytes = 0;
  return 0;
}

int fhip_sample_supported(const fhip_sample_desc *d) {
  if (!d || validate(nullptr, d) != 0)
    return 0;
  return 1;
}

int fhip_sample(fhip_ctx *ctx, const fhip_sample_desc *d, const void *logits, const void *uniform, const void *temperature,
                const void *top_k, const void *top_p, const void *min_p, void *token, void *probability, void *workspace,
                size_t workspace_bytes) {
  static const char who[] = "fhip_sample";
  FHIP_REQUIRE(ctx, ctx != nullptr, "%s: null context", who);
  if (validate(ctx, d) != 0)
    return 1;
  FHIP_REQUIRE(ctx, logits && uniform && token, "%s: null tensor pointer", who);
  FHIP_REQUIRE(ctx, (d->has_temperature != 0) == (temperature != nullptr) && (d->has_top_k != 0) == (top_k != nullptr) &&
                        (d->has_top_p != 0) == (top_p != nullptr) && (d->has_min_p != 0) == (min_p != nullptr),
               "%s: settings' pointers and the descriptor disagree", who);
  (void)workspace;
  (void)workspace_bytes;
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  SampleArgs g{};
  g.logits = logits, g.uniform = (const float *)uniform, g.temperature = (const float *)temperature;
  g.top_k = (const int32_t *)top_k, g.top_p = (const float *)top_p, g.min_p = (const float *)min_p;
  g.token = (int32_t *)token, g.probability = (float *)probability;
  g.row_s = d->logits.stride[0], g.word_s = d->logits.stride[1];
  g.rows = d->logits.dim[0], g.words = (int32_t)d->logits.dim[1], g.dtype = d->logits.dtype;
  g.one_temperature = d->temperature, g.one_top_k = d->top_k, g.one_top_p = d->top_p, g.one_min_p = d->min_p;
  fhip_note_kernel(ctx, "sample_rows");
  const int64_t most = (int64_t)ctx->num_cus * 32;
  hipLaunchKernelGGL(sample_rows_kernel, dim3((unsigned)(g.rows < most ? g.rows : most)), dim3(kThreads), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
