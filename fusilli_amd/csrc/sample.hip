// A token for each row of logits from given random numbers (fhip_sample).
//
// Words are ordered by their logits, the largest first, equal ones by their index.  What
// temperature, top-k, top-p and min-p keep is the first so many in that order, and the token is the
// first up to which the kept weights' sum exceeds uniform times all of it; so every question is for
// a prefix of the order: up to a count, up to a sum.  None of them needs the words sorted: a
// prefix ends in one value of the logits, found digit by digit from counts and sums of the words
// that share the digits above, and in one of the words that have that value, by index.
//
// Weights exp((l - m) / T) are f64 and kept as whole multiples of 2^-38 to 2^-46 of the largest, as
// many bits as leave a row's sum below 2^63: sums are exact whatever the order of the additions, so
// that every run and every way of cutting the row gives the same token.  (f32 weights would move
// one border in 10^7, and a row has 10^5 of them.)
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
  int32_t bits; // a weight of 1 is 2^bits
  // rows cut into parts
  int32_t parts, part_words;
  uint64_t *part_most; // [row][part]: largest key, then the lowest index that has it
  float *part_least;   // [row][part]: smallest logit that may be drawn
  uint64_t *sums;      // [row][part][bucket]
  uint32_t *counts;    // the same
};

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

// A row's settings.
struct Settings {
  double most, by; // the largest logit, 1 / T
  double unit;     // 2^bits
  float p, least, u;
  int k;
  bool greedy;
  __device__ __forceinline__ Settings(const SampleArgs &g, int64_t row, float largest) {
    const float t = g.temperature ? g.temperature[row] : g.one_temperature;
    k = g.top_k ? g.top_k[row] : g.one_top_k;
    p = g.top_p ? g.top_p[row] : g.one_top_p;
    least = g.min_p ? g.min_p[row] : g.one_min_p;
    u = g.uniform[row];
    most = (double)largest;
    greedy = !(t > 0.f);
    by = greedy ? 1.0 : fmax(1.0 / (double)t, 1e-300); // (T infinite: -inf times it is -inf)
    unit = (double)(1ull << g.bits);
  }
  __device__ __forceinline__ double down(float l) const { return l == (float)most ? 0.0 : ((double)l - most) * by; }
  __device__ __forceinline__ double weight(float l) const { return exp(down(l)); }
  __device__ __forceinline__ uint64_t held(float l) const {
    const double x = down(l);
    return x > -32.0 ? (uint64_t)rint(exp(x) * unit) : 0; // (exp(-32) is 2^-46.2)
  }
  // the weights' sum that top_p asks for of `all`; the sum that the token's exceeds of `kept`
  __device__ __forceinline__ uint64_t share(uint64_t all) const {
    const double x = p > 0.f ? ceil((double)p * (double)all) : 1.0;
    return x < 1.0 ? 1 : x < (double)all ? (uint64_t)x : all;
  }
  __device__ __forceinline__ uint64_t below(uint64_t kept) const {
    const double x = u > 0.f ? floor((double)u * (double)kept) : 0.0;
    const uint64_t at = x < (double)kept ? (uint64_t)x : kept;
    return at < kept ? at : kept - 1;
  }
};

// The end of a prefix: the last value that it holds, how many words have larger ones and their
// weights, and how many words of that value it takes.
struct End {
  uint32_t key;
  uint32_t count;
  uint64_t sum;
  uint32_t ties;
};

template <int NT> struct Shared {
  uint64_t sum[256];
  uint32_t count[256];
  uint32_t digit, above_count;
  uint64_t above_sum;
  uint64_t wave[NT / 64];
};

template <int NT, typename F> __device__ __forceinline__ uint64_t over_workgroup(uint64_t v, Shared<NT> &s, F join) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1)
    v = join(v, (uint64_t)__shfl_xor((unsigned long long)v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    s.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.wave[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w)
    v = join(v, s.wave[w]);
  return v;
}

// The end of the shortest prefix of items 0 .. n - 1 that holds `need` of them (by_count) or whose
// weights' sum is at least `need`; there is as much.  key_at(i): an item's key, 0 for none.  Eight
// bits at a time from the highest one in which keys differ (items of one bucket share most of
// theirs, and all additions would go to a few places).
template <int NT, typename Key, typename Held>
__device__ __forceinline__ End find_end(bool by_count, uint64_t need, int n, Shared<NT> &s, Key key_at, Held held) {
  uint32_t high = 0, low = 0; // largest key, and complement of the smallest
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint32_t key = key_at(i);
    high = key > high ? key : high;
    low = key && ~key > low ? ~key : low;
  }
  const uint64_t both = over_workgroup<NT>((uint64_t)high << 32 | low, s, [](uint64_t a, uint64_t b) {
    const uint64_t h = (a >> 32) > (b >> 32) ? a >> 32 : b >> 32;
    const uint32_t l = (uint32_t)a > (uint32_t)b ? (uint32_t)a : (uint32_t)b;
    return h << 32 | l;
  });
  high = (uint32_t)(both >> 32), low = ~(uint32_t)both;
  int left = high == low ? 0 : 32 - __builtin_clz(high ^ low); // bits in which keys differ
  uint32_t prefix = left == 32 ? 0 : high >> left << left;
  uint32_t count = 0, same = 0;
  uint64_t sum = 0;
  do {
    const int shift = left > 8 ? left - 8 : 0;
    const uint32_t above = left == 32 ? 0 : ~0u << left; // bits that the prefix has
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += NT)
      s.sum[i] = 0, s.count[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
      const uint32_t key = key_at(i);
      if (key == 0 || (key & above) != prefix)
        continue;
      const int digit = (int)((key & ~above) >> shift);
      atomicAdd(&s.count[digit], 1u);
      atomicAdd((unsigned long long *)&s.sum[digit], (unsigned long long)held(key));
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      // four digits a lane, the largest first
      const int l = threadIdx.x;
      uint32_t c[4], cs = 0;
      uint64_t w[4], ws = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = s.count[255 - 4 * l - i], w[i] = s.sum[255 - 4 * l - i];
        cs += c[i], ws += w[i];
      }
      uint32_t c0 = cs;
      uint64_t w0 = ws;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t cu = __shfl_up(c0, d);
        const uint64_t wu = __shfl_up((unsigned long long)w0, d);
        if (l >= d)
          c0 += cu, w0 += wu;
      }
      c0 += count - cs, w0 += sum - ws; // in front of this lane's
      int found = -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool here = c[i] != 0 && (by_count ? c0 + c[i] >= need : w0 + w[i] >= need);
        if (here && found < 0)
          found = i;
        if (found < 0)
          c0 += c[i], w0 += w[i];
      }
      const uint64_t hit = __builtin_amdgcn_ballot_w64(found >= 0);
      if (hit && l == __builtin_ctzll(hit))
        s.digit = (uint32_t)(255 - 4 * l - found), s.above_count = c0, s.above_sum = w0;
    }
    __syncthreads();
    prefix |= s.digit << shift;
    same = s.count[s.digit];
    count = s.above_count, sum = s.above_sum;
    left = shift;
  } while (left > 0);
  End e;
  e.key = prefix, e.count = count, e.sum = sum;
  const uint64_t each = held(prefix);
  const uint64_t ties = by_count ? need - count : need <= sum || each == 0 ? 1 : (need - sum + each - 1) / each;
  e.ties = (uint32_t)(ties < 1 ? 1 : ties > same ? same : ties);
  __syncthreads();
  return e;
}

// One row, which is read again for each digit.
template <int NT> __device__ __noinline__ void sample_row(const SampleArgs &g, int64_t row, Shared<NT> &s) {
  auto key_at = [&](int i) { return key_of(fhip_load_float(g.logits, g.dtype, row * g.row_s + i * g.word_s)); };
  auto add = [](uint64_t a, uint64_t b) { return a + b; };
  uint64_t most = 0, some = 0;
  for (int i = threadIdx.x; i < g.words; i += NT) {
    const uint32_t key = key_at(i);
    most = key > most ? key : most;
    some += key != 0;
  }
  most = over_workgroup<NT>(most, s, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
  some = over_workgroup<NT>(some, s, add);
  if (some == 0) {
    if (threadIdx.x == 0) {
      g.token[row] = -1;
      if (g.probability)
        g.probability[row] = 0.f;
    }
    return;
  }
  const Settings set(g, row, logit_of((uint32_t)most));
  auto held = [&](uint32_t key) { return set.held(logit_of(key)); };
  uint64_t kept = (uint64_t)1 << g.bits; // (greedy: the first word's weight)
  if (!set.greedy) {
    // what the first k weigh
    if (set.k > 0 && (uint64_t)set.k < some) {
      const End e = find_end<NT>(true, (uint64_t)set.k, g.words, s, key_at, held);
      kept = e.sum + e.ties * held(e.key);
    } else {
      kept = 0;
      for (int i = threadIdx.x; i < g.words; i += NT)
        if (const uint32_t key = key_at(i))
          kept += held(key);
      kept = over_workgroup<NT>(kept, s, add);
    }
    uint64_t strict = kept;
    if (set.p < 1.f) {
      const End e = find_end<NT>(false, set.share(kept), g.words, s, key_at, held);
      strict = e.sum + e.ties * held(e.key);
    }
    if (set.least > 0.f) {
      uint64_t large = 0;
      const double bound = set.least < 1.f ? (double)set.least : 1.0;
      for (int i = threadIdx.x; i < g.words; i += NT) {
        const uint32_t key = key_at(i);
        if (key && set.weight(logit_of(key)) >= bound)
          large += held(key);
      }
      large = over_workgroup<NT>(large, s, add);
      strict = large < strict ? large : strict;
    }
    kept = strict < kept ? strict : kept;
    if (set.least > 1.f)
      kept = (uint64_t)1 << g.bits;
  }
  // the first word up to which the sum is above u * kept, and its index: the `ties`-th of its value
  const End e = find_end<NT>(false, (set.greedy ? 0 : set.below(kept)) + 1, g.words, s, key_at, held);
  const End at = find_end<NT>(true, e.ties, g.words, s,
                              [&](int i) { return key_at(i) == e.key ? ~(uint32_t)i : 0u; }, [](uint32_t) { return 0ull; });
  if (threadIdx.x == 0) {
    g.token[row] = (int32_t)~at.key;
    if (g.probability)
      g.probability[row] = (float)((double)held(e.key) / (double)kept);
  }
}

// Any strides and sizes: a workgroup a row.
constexpr int kRowThreads = 512;
__global__ __launch_bounds__(kRowThreads) void sample_rows_kernel(SampleArgs g) {
  __shared__ Shared<kRowThreads> s;
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    sample_row<kRowThreads>(g, row, s);
    __syncthreads();
  }
}

// ---- rows whose words lie side by side ------------------------------------------------------
// Three steps: the largest logit; sums of weights in 1024 buckets of equal width in (m - l) / T; then
// the buckets in which the prefixes can end, their words brought together in LDS and the
// questions answered there as above.  The buckets' sums are exact, so are the prefixes.  One workgroup
// takes all steps of a row where rows fill the chip or are short; otherwise the first two are launches
// over parts of rows.
//
// Buckets cover what words have above a weight of 0, less than 32 of (m - l) / T.
constexpr int kBuckets = 1024, kThreads = 1024;
constexpr int kList = 8192; // words of the buckets in question

// N words from `at` of a row whose words lie side by side, at element alignment.
template <int DT> struct Words;
template <> struct Words<FHIP_FLOAT> {
  static constexpr int N = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float one(const void *p, int64_t at) { return ((const float *)p)[at]; }
  static __device__ __forceinline__ void load(const void *p, int64_t at, float (&v)[N]) {
    const V x = *(const V *)((const float *)p + at);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  }
};
template <typename H> struct HalfWords {
  static constexpr int N = 8;
  typedef H V __attribute__((ext_vector_type(8), aligned(2)));
  static __device__ __forceinline__ float one(const void *p, int64_t at) { return (float)((const H *)p)[at]; }
  static __device__ __forceinline__ void load(const void *p, int64_t at, float (&v)[N]) {
    const V x = *(const V *)((const H *)p + at);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = (float)x[i];
  }
};
template <> struct Words<FHIP_BFLOAT16> : HalfWords<__bf16> {};
template <> struct Words<FHIP_HALF> : HalfWords<_Float16> {};

// take(logit, index) of the words from .. to - 1 of a row
template <int DT, int NT, typename Take>
__device__ __forceinline__ void for_words(const SampleArgs &g, int64_t row, int from, int to, Take take) {
  using W = Words<DT>;
  const int64_t base = row * g.row_s;
  const int whole = from + (to - from) / W::N * W::N;
#pragma unroll 4
  for (int i = from + (int)threadIdx.x * W::N; i < whole; i += NT * W::N) {
    float v[W::N];
    W::load(g.logits, base + i, v);
#pragma unroll
    for (int e = 0; e < W::N; ++e)
      take(v[e], i + e);
  }
  for (int i = whole + (int)threadIdx.x; i < to; i += NT)
    take(W::one(g.logits, base + i), i);
}

// What is known of a row, or a part of it: its largest key and the lowest index that has it (0: no
// word may be drawn), its smallest logit that may be drawn.
struct Range {
  uint64_t most;
  float least;
  __device__ __forceinline__ float largest() const { return logit_of((uint32_t)(most >> 32)); }
};
template <int DT> __device__ __forceinline__ Range range_of(const SampleArgs &g, int64_t row, int from, int to, Shared<kThreads> &s) {
  uint64_t most = 0;
  float least = INFINITY;
  for_words<DT, kThreads>(g, row, from, to, [&](float l, int i) {
    const uint64_t x = (uint64_t)key_of(l) << 32 | ~(uint32_t)i;
    most = l > -INFINITY && x > most ? x : most;
    least = l > -INFINITY ? fminf(least, l) : least;
  });
  auto larger = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
  Range r;
  r.most = over_workgroup<kThreads>(most, s, larger);
  r.least = logit_of(0xffffffffu - (uint32_t)over_workgroup<kThreads>((uint64_t)(0xffffffffu - key_of(least)), s, larger));
  return r;
}

// A row's buckets: the first holds the largest logits.
struct Buckets {
  double most, by;
  float top;
  __device__ __forceinline__ Buckets(const Settings &set, float least) : most(set.most), top((float)set.most) {
    const double wide = -set.down(least);
    // (a little less than the range takes, so that the last word is inside)
    by = wide > 0.0 ? set.by * (kBuckets * (1.0 - 0x1p-20)) / (wide < 32.0 ? wide : 32.0) : 0.0;
  }
  __device__ __forceinline__ int of(float l) const { // kBuckets and more: none
    const double b = l == top ? 0.0 : (most - (double)l) * by;
    return b < (double)kBuckets ? (int)b : kBuckets;
  }
};

struct Sums {
  uint64_t sum[kBuckets];
  uint32_t count[kBuckets];
};
template <int DT>
__device__ __forceinline__ void sums_of(const SampleArgs &g, int64_t row, int from, int to, const Settings &set,
                                        const Buckets &buckets, bool count, Sums &s) {
  s.sum[threadIdx.x] = 0, s.count[threadIdx.x] = 0;
  __syncthreads();
  for_words<DT, kThreads>(g, row, from, to, [&](float l, int) {
    if (!(l > -INFINITY))
      return;
    const int b = buckets.of(l);
    if (b >= kBuckets)
      return;
    atomicAdd((unsigned long long *)&s.sum[b], (unsigned long long)set.held(l));
    if (count)
      atomicAdd(&s.count[b], 1u);
  });
  __syncthreads();
}

struct Draw {
  Shared<kThreads> s;
  uint64_t before[kBuckets + 1]; // weights in front of a bucket
  uint8_t asked[kBuckets];
  int located[6], filled;
  uint32_t count_before;
  uint32_t keys[kList], places[kList];
  uint16_t homes[kList];
};

// A row without a question; false: there are some.
__device__ __forceinline__ bool settled(const SampleArgs &g, int64_t row, const Range &range) {
  const float t = g.temperature ? g.temperature[row] : g.one_temperature;
  if (range.most != 0 && t > 0.f)
    return false;
  if (threadIdx.x == 0) {
    g.token[row] = range.most == 0 ? -1 : (int32_t)~(uint32_t)range.most;
    if (g.probability)
      g.probability[row] = range.most == 0 ? 0.f : 1.f;
  }
  return true;
}

// The token of a row; `mine` and `here`: weights and words of this thread's bucket.
template <int DT>
__device__ __forceinline__ void draw_row(const SampleArgs &g, int64_t row, const Settings &set, const Buckets &buckets,
                                         bool count, uint64_t mine, uint32_t here, Draw &d) {
  constexpr int NT = kThreads;
  static_assert(NT == kBuckets, "a thread a bucket");
  const int b = threadIdx.x;
  auto in_front = [&](uint64_t v) { // exclusive sums over the threads
    uint64_t x = v;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint64_t y = __shfl_up((unsigned long long)x, k);
      x += (threadIdx.x & 63) >= k ? y : 0;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63)
      d.s.wave[threadIdx.x >> 6] = x;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w)
      x += d.s.wave[w];
    return x - v;
  };
  const uint64_t start = in_front(mine);
  const uint32_t first = count ? (uint32_t)in_front(here) : 0;
  d.before[b] = start;
  if (b == NT - 1)
    d.before[kBuckets] = start + mine;
  if (b < 6)
    d.located[b] = -1;
  if (b == 0)
    d.filled = 0;
  __syncthreads();
  const uint64_t all = d.before[kBuckets];
  // which bucket holds the `need`-th unit of weight
  auto locate = [&](int slot, uint64_t need) {
    if (start < need && need <= start + mine)
      d.located[slot] = b;
  };
  // What is kept weighs between `low` and `high`, until the words are known in which a prefix ends.
  if (count && first < (uint32_t)set.k && (uint32_t)set.k <= first + here) {
    d.located[0] = b;
    d.count_before = first;
  }
  __syncthreads();
  const int by_k = d.located[0]; // (-1: fewer words than k weigh anything)
  uint64_t low = all, high = all;
  if (by_k >= 0)
    low = d.before[by_k], high = d.before[by_k + 1];
  low = low < 1 ? 1 : low;
  const bool by_p = set.p < 1.f;
  if (by_p) {
    locate(1, set.share(low));
    locate(2, set.share(high));
    __syncthreads();
    low = d.before[d.located[1]], high = d.before[d.located[2] + 1];
  }
  const bool by_least = set.least > 0.f;
  const double bound = set.least < 1.f ? (double)set.least : 1.0;
  int least_from = kBuckets, least_to = kBuckets;
  if (by_least) {
    const double at = -log(bound) / set.by * buckets.by;
    const double a = at - 1e-6, z = at + 1e-6;
    least_from = a < 0.0 ? 0 : a < (double)kBuckets ? (int)a : kBuckets;
    least_to = z < (double)kBuckets ? (int)z : kBuckets;
    if (least_from < kBuckets) {
      const uint64_t a_sum = d.before[least_from], z_sum = d.before[least_to < kBuckets ? least_to + 1 : kBuckets];
      low = a_sum < low ? a_sum : low;
      high = z_sum < high ? z_sum : high;
    }
  }
  const uint64_t one = (uint64_t)1 << g.bits; // (the largest is always kept)
  low = low < one ? one : low;
  high = high < low ? low : high;
  if (set.least > 1.f)
    low = high = one;
  locate(3, set.below(low) + 1);
  locate(4, set.below(high) + 1);
  __syncthreads();
  d.asked[b] = b == by_k || (by_p && b >= d.located[1] && b <= d.located[2]) || (b >= least_from && b <= least_to) ||
               (b >= d.located[3] && b <= d.located[4]);
  __syncthreads();
  // the words of those buckets
  for_words<DT, NT>(g, row, 0, g.words, [&](float l, int i) {
    if (!(l > -INFINITY))
      return;
    const int home = buckets.of(l);
    if (home >= kBuckets || !d.asked[home])
      return;
    const int to = atomicAdd(&d.filled, 1);
    if (to < kList)
      d.keys[to] = key_of(l), d.places[to] = (uint32_t)i, d.homes[to] = (uint16_t)home;
  });
  __syncthreads();
  const int n = d.filled;
  if (n > kList) { // (many equal logits)
    sample_row<NT>(g, row, d.s);
    return;
  }
  auto held = [&](uint32_t key) { return set.held(logit_of(key)); };
  auto of_bucket = [&](int home) { return [&, home](int i) { return d.homes[i] == home ? d.keys[i] : 0u; }; };
  auto bucket_of = [&](uint64_t need) {
    __syncthreads();
    locate(5, need);
    __syncthreads();
    return d.located[5];
  };
  uint64_t kept = all;
  if (by_k >= 0) {
    const End e = find_end<NT>(true, (uint64_t)set.k - d.count_before, n, d.s, of_bucket(by_k), held);
    kept = d.before[by_k] + e.sum + e.ties * held(e.key);
  }
  uint64_t strict = kept;
  if (by_p) {
    const uint64_t need = set.share(kept);
    const int home = bucket_of(need);
    const End e = find_end<NT>(false, need - d.before[home], n, d.s, of_bucket(home), held);
    strict = d.before[home] + e.sum + e.ties * held(e.key);
  }
  if (by_least && least_from < kBuckets) {
    uint64_t large = 0;
    for (int i = threadIdx.x; i < n; i += NT)
      if (d.homes[i] >= least_from && d.homes[i] <= least_to && set.weight(logit_of(d.keys[i])) >= bound)
        large += held(d.keys[i]);
    large = d.before[least_from] + over_workgroup<NT>(large, d.s, [](uint64_t a, uint64_t c) { return a + c; });
    strict = large < strict ? large : strict;
  }
  kept = strict < kept ? strict : kept;
  if (set.least > 1.f)
    kept = one;
  const uint64_t need = set.below(kept) + 1;
  const int home = bucket_of(need);
  const End e = find_end<NT>(false, need - d.before[home], n, d.s, of_bucket(home), held);
  const End at = find_end<NT>(true, e.ties, n, d.s, [&](int i) { return d.keys[i] == e.key ? ~d.places[i] : 0u; },
                              [](uint32_t) { return 0ull; });
  if (b == 0) {
    g.token[row] = (int32_t)~at.key;
    if (g.probability)
      g.probability[row] = (float)((double)held(e.key) / (double)kept);
  }
}

__device__ __forceinline__ bool counts_words(const SampleArgs &g, const Settings &set) { return set.k > 0 && set.k < g.words; }

// A workgroup a row.
template <int DT> __global__ __launch_bounds__(kThreads) void sample_whole_kernel(SampleArgs g) {
  __shared__ Draw d;
  __shared__ Sums sums;
  const int64_t row = blockIdx.x;
  const Range range = range_of<DT>(g, row, 0, g.words, d.s);
  if (settled(g, row, range))
    return;
  const Settings set(g, row, range.largest());
  const Buckets buckets(set, range.least);
  const bool count = counts_words(g, set);
  sums_of<DT>(g, row, 0, g.words, set, buckets, count, sums);
  draw_row<DT>(g, row, set, buckets, count, sums.sum[threadIdx.x], sums.count[threadIdx.x], d);
}

template <int DT> __global__ __launch_bounds__(kThreads) void sample_most_kernel(SampleArgs g) {
  __shared__ Shared<kThreads> s;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  const int from = part * g.part_words, to = from + g.part_words < g.words ? from + g.part_words : g.words;
  const Range r = range_of<DT>(g, row, from, to, s);
  if (threadIdx.x == 0) {
    g.part_most[row * g.parts + part] = r.most;
    g.part_least[row * g.parts + part] = r.least;
  }
}

__device__ __forceinline__ Range range_of_parts(const SampleArgs &g, int64_t row) {
  Range r{0, INFINITY};
  for (int p = 0; p < g.parts; ++p) {
    const uint64_t m = g.part_most[row * g.parts + p];
    r.most = m > r.most ? m : r.most;
    r.least = fminf(r.least, g.part_least[row * g.parts + p]);
  }
  return r;
}

template <int DT> __global__ __launch_bounds__(kThreads) void sample_sums_kernel(SampleArgs g) {
  __shared__ Sums sums;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  const Range range = range_of_parts(g, row);
  if (range.most == 0)
    return;
  const Settings set(g, row, range.largest());
  if (set.greedy)
    return;
  const Buckets buckets(set, range.least);
  const bool count = counts_words(g, set);
  const int from = part * g.part_words, to = from + g.part_words < g.words ? from + g.part_words : g.words;
  sums_of<DT>(g, row, from, to, set, buckets, count, sums);
  const int64_t at = (row * g.parts + part) * kBuckets + threadIdx.x;
  g.sums[at] = sums.sum[threadIdx.x];
  if (count)
    g.counts[at] = sums.count[threadIdx.x];
}

template <int DT> __global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs g) {
  __shared__ Draw d;
  const int64_t row = blockIdx.x;
  const Range range = range_of_parts(g, row);
  if (settled(g, row, range))
    return;
  const Settings set(g, row, range.largest());
  const Buckets buckets(set, range.least);
  const bool count = counts_words(g, set);
  uint64_t mine = 0;
  uint32_t here = 0;
  for (int p = 0; p < g.parts; ++p) {
    const int64_t at = (row * g.parts + p) * kBuckets + threadIdx.x;
    mine += g.sums[at];
    if (count)
      here += g.counts[at];
  }
  draw_row<DT>(g, row, set, buckets, count, mine, here, d);
}

// How rows are cut: parts that fill the chip, of 4096 words at least (one part: a workgroup a row).
struct Cut {
  int parts, words;
  Cut(int64_t rows, int64_t row_words) {
    int64_t n = rows >= 128 ? 1 : 512 / rows;
    const int64_t most = (row_words + 4095) / 4096;
    n = n < most ? n : most;
    n = n < 32 ? n : 32;
    words = (int)(((row_words + n - 1) / n + 7) / 8 * 8);
    parts = (int)((row_words + words - 1) / words);
  }
};

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

static bool side_by_side(const fhip_sample_desc &d) { return d.logits.stride[1] == 1 || d.logits.dim[1] == 1; }
// Where things lie in the workspace, which begins with the parts' largest logits.
struct Places {
  size_t least, sums, counts, bytes;
};
static Places places_of(const fhip_sample_desc &d) {
  Places p{};
  const Cut c(d.logits.dim[0], d.logits.dim[1]);
  if (!side_by_side(d) || c.parts == 1)
    return p;
  const size_t n = (size_t)d.logits.dim[0] * (size_t)c.parts;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p.least = up(n * 8);
  p.sums = p.least + up(n * 4);
  p.counts = p.sums + n * kBuckets * 8;
  p.bytes = p.counts + n * kBuckets * 4;
  return p;
}

template <int DT> static int launch(fhip_ctx *ctx, const SampleArgs &g) {
  if (g.parts == 1) {
    hipLaunchKernelGGL(sample_whole_kernel<DT>, dim3((unsigned)g.rows), dim3(kThreads), 0, ctx->stream, g);
  } else { // (fewer than 128 rows)
    const dim3 grid((unsigned)g.parts, (unsigned)g.rows);
    hipLaunchKernelGGL(sample_most_kernel<DT>, grid, dim3(kThreads), 0, ctx->stream, g);
    hipLaunchKernelGGL(sample_sums_kernel<DT>, grid, dim3(kThreads), 0, ctx->stream, g);
    hipLaunchKernelGGL(sample_draw_kernel<DT>, dim3((unsigned)g.rows), dim3(kThreads), 0, ctx->stream, g);
  }
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

extern "C" {

int fhip_sample_workspace_size(const fhip_sample_desc *d, size_t *bytes) {
  FHIP_REQUIRE(nullptr, d && bytes, "fhip_sample_workspace_size: null");
  if (validate(nullptr, d) != 0)
    return 1;
  *bytes = places_of(*d).bytes;
  return 0;
}

int fhip_sample_supported(const fhip_sample_desc *d) {
  if (!d || validate(nullptr, d) != 0)
    return 0;
  return side_by_side(*d) ? 2 : 1;
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
  const Places at = places_of(*d);
  if (at.bytes)
    FHIP_REQUIRE(ctx, workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= at.bytes,
                 "%s: needs %zu bytes of 256-byte aligned workspace", who, at.bytes);
  FHIP_HIP_CHECK(ctx, hipSetDevice(ctx->device));
  SampleArgs g{};
  g.logits = logits, g.uniform = (const float *)uniform, g.temperature = (const float *)temperature;
  g.top_k = (const int32_t *)top_k, g.top_p = (const float *)top_p, g.min_p = (const float *)min_p;
  g.token = (int32_t *)token, g.probability = (float *)probability;
  g.row_s = d->logits.stride[0], g.word_s = d->logits.stride[1];
  g.rows = d->logits.dim[0], g.words = (int32_t)d->logits.dim[1], g.dtype = d->logits.dtype;
  g.one_temperature = d->temperature, g.one_top_k = d->top_k, g.one_top_p = d->top_p, g.one_min_p = d->min_p;
  g.bits = 0;
  while (g.bits < 46 && ((int64_t)g.words << (g.bits + 1)) <= (1ll << 62))
    ++g.bits;
  if (side_by_side(*d) && g.rows < (1 << 21)) { // (a grid's threads are a number below 2^32)
    const Cut c(g.rows, g.words);
    g.parts = c.parts, g.part_words = c.words;
    char *w = (char *)workspace;
    g.part_most = (uint64_t *)w, g.part_least = (float *)(w + at.least);
    g.sums = (uint64_t *)(w + at.sums), g.counts = (uint32_t *)(w + at.counts);
    fhip_note_kernel(ctx, "sample parts=%d", c.parts);
    switch (g.dtype) {
    case FHIP_FLOAT: return launch<FHIP_FLOAT>(ctx, g);
    case FHIP_BFLOAT16: return launch<FHIP_BFLOAT16>(ctx, g);
    default: return launch<FHIP_HALF>(ctx, g);
    }
  }
  fhip_note_kernel(ctx, "sample_rows");
  const int64_t most = (int64_t)ctx->num_cus * 32;
  hipLaunchKernelGGL(sample_rows_kernel, dim3((unsigned)(g.rows < most ? g.rows : most)), dim3(kRowThreads), 0, ctx->stream, g);
  FHIP_HIP_CHECK(ctx, hipGetLastError());
  return 0;
}

} // extern "C"
