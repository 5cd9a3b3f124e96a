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

#include <type_traits>

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
  unsigned long long *sums; // [row][bucket], cleared by the first launch
  uint32_t *counts;         // the same
  uint32_t *filled, *arrived; // [row]: words of the buckets in question, parts that have written theirs; cleared too
  unsigned long long *list;   // [row][kList]: such a word's index, logit
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

// A row's settings as they are given.  All loads at once, those of absent vectors from the uniform
// numbers: behind a branch each would wait for memory by itself, a microsecond every time.
struct Asked {
  float t, p, least, u;
  int k;
  __device__ __forceinline__ Asked(const SampleArgs &g, int64_t row) {
    const float *const vt = g.temperature ? g.temperature : g.uniform, *const vp = g.top_p ? g.top_p : g.uniform;
    const float *const vl = g.min_p ? g.min_p : g.uniform;
    const int32_t *const vk = g.top_k ? g.top_k : (const int32_t *)g.uniform;
    t = vt[row], p = vp[row], least = vl[row], k = vk[row], u = g.uniform[row];
    t = g.temperature ? t : g.one_temperature;
    k = g.top_k ? k : g.one_top_k;
    p = g.top_p ? p : g.one_top_p;
    least = g.min_p ? least : g.one_min_p;
  }
};

// 1 / x, good to two steps or so of f64 (x = 0: infinity or NaN; infinite: 0 or NaN): a seed that is good to
// 2^-24 and two of Newton's steps.
__device__ __forceinline__ double reciprocal(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = __builtin_fma(y, __builtin_fma(-x, y, 1.0), y);
  return __builtin_fma(y, __builtin_fma(-x, y, 1.0), y);
}

// (m - l) / T from which on no weight is held.
constexpr double kFar = 33.0;

struct Settings : Asked {
  double most, by;  // the largest logit, 1 / T
  double by2;       // log2(e) / T
  float top;        // the largest logit
  int bits;
  bool greedy;
  __device__ __forceinline__ Settings(const SampleArgs &g, const Asked &asked, float largest) : Asked(asked) {
    most = (double)largest;
    greedy = !(t > 0.f);
    // (T infinite: NaN here, and 1e-100, with which -inf is -inf, any other difference times it less than 2^-200 and
    // the smallest one's reciprocal a number)
    by = greedy ? 1.0 : fmax(reciprocal((double)t), 1e-100);
    by2 = by * 1.44269504088896340736;
    top = largest;
    bits = g.bits;
  }
  // The weight of a logit that is finite like the largest and less than 64 T below it, times 2^up.  2^x
  // with x = n + f, |f| at most 1/2: a polynomial of degree 10 through 1 at 0 that meets 2^f at the zeros of a
  // Chebyshev polynomial (6e-16 of it off at most).  Adding 3 * 2^51 rounds x to its n, which stands in the
  // sum's low bits and is added to the exponent from there: f64's own rint, conversion and ldexp are
  // issued at a quarter of the rate.
  __device__ __forceinline__ double near_weight(float l, int up) const {
    const double off = (double)l - most, whole = __builtin_fma(off, by2, 0x1.8p52);
    const double f = __builtin_fma(off, by2, 0x1.8p52 - whole);
    // (the constants keep their registers: in C++ each becomes a copy and an instruction that overwrites it)
    auto step = [&](double y, double c) {
      double r;
      asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(y), "v"(f), "s"(c));
      return r;
    };
    double y = step(7.0709662925771758e-09, 1.0205905366447884e-07);
    y = step(y, 1.3215451705400571e-06);
    y = step(y, 1.5252672925113478e-05);
    y = step(y, 1.5403530424618647e-04);
    y = step(y, 1.3333558200794100e-03);
    y = step(y, 9.6181291076188023e-03);
    y = step(y, 5.5504108664651677e-02);
    y = step(y, 2.4022650695910075e-01);
    y = step(y, 6.9314718055994617e-01);
    y = __builtin_fma(y, f, 1.0);
    const uint64_t bits_of = __builtin_bit_cast(uint64_t, y);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, whole) + (uint32_t)up;
    return __builtin_bit_cast(double, (uint64_t)((uint32_t)(bits_of >> 32) + (n << 20)) << 32 | (uint32_t)bits_of);
  }
  __device__ __forceinline__ double weight(float l) const {
    return l == top ? 1.0 : ((double)l - most) * by > -40.0 ? near_weight(l, 0) : 0.0;
  }
  // The weight in units of 2^-bits, rounded: 2^52 on top leaves it in the low bits.
  __device__ __forceinline__ uint64_t held_near(float l) const {
    return __builtin_bit_cast(uint64_t, near_weight(l, bits) + 0x1p52) & ((1ull << 52) - 1);
  }
  // The same of any.  0 beyond kFar, where held_near is 0 as well (from exp(-32.58) = 2^-47 on): whichever of the
  // two a kernel asks, sums and the words that they are made of agree, also where buckets end a rounding off kFar.
  __device__ __forceinline__ uint64_t held(float l) const {
    return l == top ? 1ull << bits : ((double)l - most) * by > -kFar ? held_near(l) : 0;
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
  uint32_t ties, same; // (all words of that value: those of the items that were asked for)
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
  e.same = same;
  const uint64_t each = held(prefix);
  const uint64_t ties = by_count ? need - count : need <= sum || each == 0 ? 1 : (need - sum + each - 1) / each;
  e.ties = (uint32_t)(ties < 1 ? 1 : ties > same ? same : ties);
  __syncthreads();
  return e;
}

// One row, which is read again for each digit.  (Inlined: a call would give its callers a stack, which
// costs 3 us or so a launch, and its registers, with which half as many wavefronts fit.)
template <int NT> __device__ __forceinline__ void sample_row(const SampleArgs &g, int64_t row, Shared<NT> &s) {
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
  const Settings set(g, Asked(g, row), logit_of((uint32_t)most));
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
// the buckets in which the prefixes can end, their words brought together in LDS, put in order there, and
// every question answered by the word whose sum says so.  The buckets' sums are exact, so are the prefixes.
// One workgroup takes all steps of a row where rows fill the chip or are short; otherwise they are three
// launches over parts of rows, the last part of a row answering.
//
// Buckets cover what words have above a weight of 0, less than 33 of (m - l) / T (kFar).  Which of them matter one
// wavefront finds, without a barrier: sixteen that execute the same few hundred instructions
// between barriers take three times as long.
//
// Bound by memory (three walks, of which caches feed the last two) and by f64 arithmetic, 30 instructions a
// word, where rows are many: f32 256 x 131072, 134 MB, 93 to 97 us, of it 28 for the largest logits (4.8 TB/s), 39 for
// the sums (20 without the exponentials), 16 for bringing together; by what runs once where they are few: code
// that no cache holds yet, loads that wait for each other, three launches.  1 x 65536 17 to 19 us, bf16 48 x 131072
// 39 to 40 us (launches 6.6, 12 and 21, of which putting 1300 words of its flattest row in order takes 10), f16
// 7 x 100003 24 to 27, f32 25 x 536 10.
constexpr int kBuckets = 1024;
constexpr int kThreads = 1024; // of the launches over parts
// How many words of the buckets in question NT threads hold, and how many of them they sort.
constexpr int list_of(int nt) { return nt == 64 ? 1024 : nt == 1024 ? 8192 : 4096; }
constexpr int kOwn = 4; // of them in a thread
constexpr int sorted_of(int nt) { return kOwn * nt; }
constexpr int kDraw = 512; // threads of the launch that draws, if it is one of its own
constexpr int kRanked = 256; // up to so many words a place is counted
constexpr int kList = 8192; // words that its workgroups hand over, of a row

// N words from `at` of a row whose words lie side by side, at element alignment.
template <typename E, int COUNT> struct WordsOf {
  static constexpr int N = COUNT;
  typedef E V __attribute__((ext_vector_type(COUNT), aligned(sizeof(E))));
  static __device__ __forceinline__ float one(const void *p, int64_t at) { return (float)((const E *)p)[at]; }
  static __device__ __forceinline__ V load(const void *p, int64_t at) { return *(const V *)((const E *)p + at); }
};
template <int DT> struct Words;
template <> struct Words<FHIP_FLOAT> : WordsOf<float, 4> {};
template <> struct Words<FHIP_BFLOAT16> : WordsOf<__bf16, 8> {};
template <> struct Words<FHIP_HALF> : WordsOf<_Float16, 8> {};

// take(logits, first index) of the words from .. to - 1 of a row, N of them at a time (-inf where
// fewer are left), with U loads on their way.
template <int NT, int DT, int U, typename Take>
__device__ __forceinline__ void for_words(const SampleArgs &g, int64_t row, int from, int to, Take take) {
  using W = Words<DT>;
  constexpr int STEP = NT * W::N;
  const int64_t base = row * g.row_s;
  const int whole = from + (to - from) / W::N * W::N, last = whole - W::N;
  const int first = from + (int)threadIdx.x * W::N;
  typename W::V raw[U];
  auto fetch = [&](int u, int i) { raw[u] = W::load(g.logits, base + (i < last ? i : last)); };
  if (last >= from) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      fetch(u, first + u * STEP);
#pragma clang loop unroll(disable)
    for (int i = first; i < whole; i += U * STEP) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[W::N];
#pragma unroll
        for (int e = 0; e < W::N; ++e)
          v[e] = (float)raw[u][e];
        fetch(u, i + (u + U) * STEP);
        if (u == 0 || i + u * STEP < whole)
          take(v, i + u * STEP);
      }
    }
  }
  if (whole + (int)threadIdx.x < to) { // (fewer than a vector)
    float v[W::N];
    v[0] = W::one(g.logits, base + whole + threadIdx.x);
#pragma unroll
    for (int e = 1; e < W::N; ++e)
      v[e] = -INFINITY;
    take(v, whole + (int)threadIdx.x);
  }
}

// Sums over the lanes up to each, and the largest value of a wavefront.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t from_lane(uint32_t v) { // (0 where there is none)
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 15, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t from_lane(uint64_t v) {
  return (uint64_t)from_lane<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | from_lane<CTRL, ROWS>((uint32_t)v);
}
template <typename T, typename F> __device__ __forceinline__ T up_to_lane(T v, F join) {
  v = join(v, from_lane<0x111, 15>(v)); // from 1, 2, 4 and 8 lanes below in a row of 16
  v = join(v, from_lane<0x112, 15>(v));
  v = join(v, from_lane<0x114, 15>(v));
  v = join(v, from_lane<0x118, 15>(v));
  v = join(v, from_lane<0x142, 10>(v)); // a row's last lane to the next row, the first half's to the second
  v = join(v, from_lane<0x143, 12>(v));
  return v;
}
template <typename T> __device__ __forceinline__ T sum_up_to_lane(T v) {
  return up_to_lane(v, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// All lanes' values joined (a value joined with itself is the same).
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T lane_or_own(T v) {
  const int own = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(own, own, CTRL, ROWS, 15, false));
}
template <typename T, typename F> __device__ __forceinline__ T joined_lanes(T v, F join) {
  v = join(v, lane_or_own<0x111, 15>(v));
  v = join(v, lane_or_own<0x112, 15>(v));
  v = join(v, lane_or_own<0x114, 15>(v));
  v = join(v, lane_or_own<0x118, 15>(v));
  v = join(v, lane_or_own<0x142, 10>(v));
  v = join(v, lane_or_own<0x143, 12>(v));
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
template <typename T> __device__ __forceinline__ T largest_of_wave(T v) {
  return of_lane(up_to_lane(v, [](T a, T b) { return a > b ? a : b; }), 63);
}
// (a wavefront's LDS accesses keep their order; this keeps the compiler from changing it)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// What is known of a row, or a part of it: its largest key and the complement of the lowest index that has
// it (0: no word may be drawn), its smallest logit that may be drawn.
struct Range {
  uint64_t most;
  float least;
  __device__ __forceinline__ float largest() const { return logit_of((uint32_t)(most >> 32)); }
};
template <int NT> struct RangeRoom {
  float top[NT / 64], least[NT / 64];
  uint32_t place[NT / 64];
};
// The same of 64 values that lanes hold: a largest value and the lowest place that has it.
__device__ __forceinline__ Range range_of_lanes(float top, uint32_t place, float least) {
  auto larger = [](float a, float b) { return fmaxf(a, b); };
  const float most = joined_lanes(top, larger);
  const uint32_t first = joined_lanes(top == most ? place : ~0u, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
  Range r;
  r.most = most > -INFINITY ? (uint64_t)key_of(most) << 32 | ~first : 0;
  r.least = joined_lanes(least, [](float a, float b) { return fminf(a, b); });
  return r;
}
template <int NT, int DT>
__device__ __forceinline__ Range range_of(const SampleArgs &g, int64_t row, int from, int to, RangeRoom<NT> &room) {
  using W = Words<DT>;
  // (a thread's indices ascend: a later word has to be larger)
  float top = -INFINITY, least = INFINITY;
  int place = 0;
  for_words<NT, DT, NT == 64 ? 2 : 4>(g, row, from, to, [&](const float(&v)[W::N], int i) {
#pragma unroll
    for (int e = 0; e < W::N; ++e) {
      place = v[e] > top ? i + e : place;
      top = v[e] > top ? v[e] : top;
      least = v[e] > -INFINITY && v[e] < least ? v[e] : least;
    }
  });
  Range r = range_of_lanes(top, (uint32_t)place, least);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) {
      room.top[threadIdx.x >> 6] = r.most ? r.largest() : -INFINITY;
      room.place[threadIdx.x >> 6] = ~(uint32_t)r.most;
      room.least[threadIdx.x >> 6] = r.least;
    }
    __syncthreads();
    const int w = threadIdx.x & (NT / 64 - 1);
    r = range_of_lanes(room.top[w], room.place[w], room.least[w]);
  }
  return r;
}

// A row's buckets: the first holds the largest logits.  In f32, whose differences and products keep the
// order; halves, as a difference may be twice the largest number.  (Of rows whose largest logit is finite.)
struct Buckets {
  float half, by;
  float a_unit; // buckets to a unit of (m - l) / T
  __device__ __forceinline__ Buckets(const Settings &set, float least) : half(0.5f * set.top) {
    const double range = (set.most - (double)least) * set.by;
    // (a little less than the range takes, so that the last word is inside for all roundings)
    const double unit = range > 0.0 ? kBuckets * (1.0 - 0x1p-20) * reciprocal(range < kFar ? range : kFar) : 0.0;
    const double x = 2.0 * set.by * unit;
    by = x < 3.0e38 ? (float)x : 3.0e38f;
    a_unit = unit < 3.0e38 ? (float)unit : 3.0e38f;
  }
  __device__ __forceinline__ int of(float l) const { // kBuckets: none
    return (int)fminf((half - 0.5f * l) * by, (float)kBuckets); // (NaN, -inf: none)
  }
};
// Where a bucket lies in LDS: a lane's sixteen in a row, lanes on banks of their own.
__device__ __forceinline__ int bucket_place(int b) { return b + (b >> 4); }
constexpr int kPlaces = kBuckets + kBuckets / 16 + 1;
constexpr int kNowhere = kPlaces, kAllPlaces = kPlaces + 64; // what is in none, by lane

struct Sums {
  unsigned long long sum[kAllPlaces];
  uint32_t count[kAllPlaces];
};
template <int NT, int DT>
__device__ __forceinline__ void sums_of(const SampleArgs &g, int64_t row, int from, int to, const Settings &set,
                                        const Buckets &buckets, bool count, Sums &s) {
  using W = Words<DT>;
  for (int i = threadIdx.x; i < kPlaces; i += NT)
    s.sum[i] = 0, s.count[i] = 0;
  __syncthreads();
  for_words<NT, DT, 1>(g, row, from, to, [&](const float(&v)[W::N], int) {
#pragma unroll
    for (int e = 0; e < W::N; ++e) {
      const int b = buckets.of(v[e]);
      const int at = b < kBuckets ? bucket_place(b) : kNowhere + (int)(threadIdx.x & 63);
      atomicAdd(&s.sum[at], (unsigned long long)set.held_near(v[e]));
      if (count)
        atomicAdd(&s.count[at], 1u);
    }
  });
  __syncthreads();
}

struct Bins {
  uint64_t sum[256];
  uint32_t count[256];
};
// What is known of a row when its buckets' sums are.
struct Front {
  uint64_t before[kPlaces]; // weights in front of a bucket
  uint32_t first[kPlaces];  // words in front of it
  uint64_t all;
  float floor; // no word in question is smaller
  int by_k, least_from, least_to;
};
template <int NT> struct Draw {
  union {
    Bins bins;
    Shared<NT> whole; // of a row that does not fit the list
  };
  Front f;
  uint32_t asked[kBuckets / 32 + 1]; // a bit a bucket (the last: none)
  uint64_t kept[3]; // what weighs no more than top_k, top_p and min_p keep
  int filled;
  uint32_t high, low, items; // largest key, complement of the smallest; how many
  End end;
  union {
    struct {
      float logits[list_of(NT)];
      uint32_t places[list_of(NT)];
    };
    alignas(16) double swap[2][sorted_of(NT)]; // (of words that registers hold)
  };
};

// find_end above over the list.  (d.high, d.low and d.items are 0 before and after.)
template <int NT, typename Key, typename Held>
__device__ __forceinline__ End list_end(bool by_count, uint64_t need, int n, Draw<NT> &d, Key key_at, Held held) {
  const int t = threadIdx.x, l = t & 63;
  auto clear = [&] {
    for (int i = t; i < 256; i += NT)
      d.bins.sum[i] = 0, d.bins.count[i] = 0;
  };
  uint32_t high = 0, low = 0, items = 0;
  for (int i = t; i - l < n; i += NT) {
    const uint32_t key = i < n ? key_at(i) : 0;
    high = key > high ? key : high;
    low = key && ~key > low ? ~key : low;
    items += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key != 0));
  }
  if (items) {
    high = largest_of_wave<uint32_t>(high), low = largest_of_wave<uint32_t>(low);
    if (l == 0)
      atomicMax(&d.high, high), atomicMax(&d.low, low), atomicAdd(&d.items, items);
  }
  clear();
  __syncthreads();
  high = d.high, low = ~d.low, items = d.items;
  int left = high == low ? 0 : 32 - __builtin_clz(high ^ low); // bits in which keys differ
  uint32_t prefix = left == 32 ? 0 : high >> left << left;
  End e{prefix, 0, 0, items, 0};
  if (left == 0) { // (equal ones: nothing to search)
    __syncthreads();
    if (t == 0)
      d.high = d.low = d.items = 0;
  }
  while (left > 0) {
    const int shift = left > 8 ? left - 8 : 0;
    const uint32_t above = left == 32 ? 0 : ~0u << left; // bits that the prefix has
    for (int i = t; i < n; i += NT) {
      const uint32_t key = key_at(i);
      if (key == 0 || (key & above) != e.key)
        continue;
      const int digit = (int)((key & ~above) >> shift);
      atomicAdd(&d.bins.count[digit], 1u);
      atomicAdd((unsigned long long *)&d.bins.sum[digit], (unsigned long long)held(key));
    }
    __syncthreads();
    if (t < 64) {
      // (four digits a lane, the largest first)
      uint32_t c[4], cs = 0;
      uint64_t w[4], ws = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = d.bins.count[255 - 4 * l - i], w[i] = d.bins.sum[255 - 4 * l - i];
        cs += c[i], ws += w[i];
      }
      uint32_t c0 = e.count + sum_up_to_lane(cs) - cs; // in front of this lane's
      uint64_t w0 = e.sum + sum_up_to_lane(ws) - ws;
      int found = -1;
      uint32_t own = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool here = c[i] != 0 && (by_count ? c0 + c[i] >= need : w0 + w[i] >= need);
        if (here && found < 0)
          found = i, own = c[i];
        if (found < 0)
          c0 += c[i], w0 += w[i];
      }
      const uint64_t hit = __builtin_amdgcn_ballot_w64(found >= 0);
      if (l == (hit ? __builtin_ctzll(hit) : 0))
        d.end = End{e.key | (uint32_t)(255 - 4 * l - (found < 0 ? 0 : found)) << shift, c0, w0, own, 0};
      if (l == 0)
        d.high = d.low = d.items = 0;
    }
    __syncthreads();
    e = d.end;
    left = shift;
    if (left > 0) {
      clear();
      __syncthreads();
    }
  }
  const uint32_t same = e.same = e.ties;
  const uint64_t each = held(e.key);
  const uint64_t ties = by_count ? need - e.count : need <= e.sum || each == 0 ? 1 : (need - e.sum + each - 1) / each;
  e.ties = (uint32_t)(ties < 1 ? 1 : ties > same ? same : ties);
  return e;
}

// Rows of no word and greedy ones have none; those whose largest logit is infinite and those at a temperature below
// 2^-90 go to sample_row.  (Further down f32 may have no number for Buckets::by, which is capped; from 2^-90 on it is
// where all words are within 6.8e-36 of the largest, hence 2^-26 of a temperature: min_p below 1 keeps them all.)
constexpr float kColdest = 0x1p-90f;
__device__ __forceinline__ bool has_questions(const Range &range, float t) {
  return range.most != 0 && t >= kColdest && range.largest() < INFINITY;
}
// Does a row without questions; false: it has some.
template <int NT>
__device__ __forceinline__ bool settled(const SampleArgs &g, int64_t row, const Range &range, float t, Shared<NT> &s) {
  if (has_questions(range, t))
    return false;
  if (range.most != 0 && t > 0.f) {
    sample_row<NT>(g, row, s);
    return true;
  }
  if (threadIdx.x == 0) {
    g.token[row] = range.most == 0 ? -1 : (int32_t)~(uint32_t)range.most;
    if (g.probability)
      g.probability[row] = range.most == 0 ? 0.f : 1.f;
  }
  return true;
}

// Where a sum ends, by a wavefront: of a lane's sixteen buckets and of all.
struct Locator {
  const Front &f;
  uint64_t start, end;
  // which bucket holds the `need`-th unit of weight (1 .. all)
  __device__ __forceinline__ int operator()(uint64_t need) const {
    const int l = threadIdx.x & 63;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(start < need && need <= end);
    const int lane = hit ? __builtin_ctzll(hit) : 0;
    const uint64_t front = __builtin_amdgcn_ballot_w64(l < 16 && f.before[lane * 17 + (l & 15)] < need);
    return lane * 16 + (front ? __builtin_popcountll(front) - 1 : 0);
  }
  __device__ __forceinline__ uint64_t start_of(int b) const { return f.before[bucket_place(b)]; }
  __device__ __forceinline__ uint64_t end_of(int b, uint64_t all) const {
    return b + 1 < kBuckets ? f.before[bucket_place(b + 1)] : all;
  }
};

__device__ __forceinline__ double least_bound(const Settings &set) { return set.least < 1.f ? (double)set.least : 1.0; }

// A lane's sixteen buckets.
struct Sixteen {
  uint64_t w[16];
  uint32_t c[16];
  template <typename Sum, typename Count> __device__ __forceinline__ void load(const Sum *sums, const Count *counts) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      w[i] = sums[i], c[i] = counts[i]; // (0 where they are not asked for)
  }
};

// The buckets in question, by the first wavefront.
template <int NT>
__device__ __forceinline__ void ask_buckets(const Settings &set, const Buckets &buckets, bool count, const Sixteen &own,
                                            Draw<NT> &d) {
  const int l = threadIdx.x;
  const uint64_t one = (uint64_t)1 << set.bits; // (the largest is always kept)
  const uint64_t(&w)[16] = own.w;
  const uint32_t(&c)[16] = own.c;
  uint64_t ws = 0;
  uint32_t cs = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    ws += w[i], cs += c[i];
  Locator locate{d.f, 0, sum_up_to_lane(ws)};
  locate.start = locate.end - ws;
  const uint64_t all = of_lane(locate.end, 63);
  const uint32_t words_end = sum_up_to_lane(cs);
  uint64_t at = locate.start;
  uint32_t words = words_end - cs;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    d.f.before[l * 17 + i] = at, d.f.first[l * 17 + i] = words;
    at += w[i], words += c[i];
  }
  if (l <= kBuckets / 32)
    d.asked[l] = 0;
  if (l == 0)
    d.filled = 0, d.high = 0, d.low = 0, d.items = 0;
  wave_fence();
  int lowest = 0; // bucket in question
  auto ask = [&](int from, int to) { // (few, or one range of many)
    lowest = to > lowest ? to : lowest;
    for (int i = from + l; i <= to; i += 64)
      atomicOr(&d.asked[i >> 5], 1u << (i & 31));
  };
  // What is kept weighs between `low` and `high`, until the words are known in which a prefix ends.
  uint64_t low = all, high = all;
  int by_k = -1, least_from = kBuckets, least_to = kBuckets;
  const uint32_t k = (uint32_t)set.k;
  const uint64_t hit = __builtin_amdgcn_ballot_w64(count && words_end - cs < k && k <= words_end);
  if (hit) { // (otherwise fewer words than k weigh anything)
    const int lane = __builtin_ctzll(hit);
    const uint64_t front = __builtin_amdgcn_ballot_w64(l < 16 && d.f.first[lane * 17 + (l & 15)] < k);
    by_k = lane * 16 + __builtin_popcountll(front) - 1;
    low = locate.start_of(by_k), high = locate.end_of(by_k, all);
    ask(by_k, by_k);
  }
  low = low < 1 ? 1 : low;
  if (set.p < 1.f) {
    const int a = locate(set.share(low)), z = locate(set.share(high));
    ask(a, z);
    low = locate.start_of(a), high = locate.end_of(z, all);
  }
  if (set.least > 0.f) {
    // (the logarithm is good to 2^-21 and 2^-21 of itself; buckets are of f32, a few roundings: less than a
    // thousandth of one)
    const float edge = -0.69314718f * __builtin_amdgcn_logf((float)least_bound(set));
    const float a = edge * (1.f - 0x1p-20f) * buckets.a_unit - buckets.a_unit * 0x1p-20f - 2e-3f;
    const float z = edge * (1.f + 0x1p-20f) * buckets.a_unit + buckets.a_unit * 0x1p-20f + 2e-3f;
    least_from = !(a > 0.f) ? 0 : a < (float)kBuckets ? (int)a : kBuckets; // (one bucket for all: 0)
    least_to = !(z > 0.f) ? 0 : z < (float)kBuckets ? (int)z : kBuckets - 1;
    if (least_from < kBuckets) {
      ask(least_from, least_to);
      const uint64_t a_sum = locate.start_of(least_from), z_sum = locate.end_of(least_to, all);
      low = a_sum < low ? a_sum : low;
      high = z_sum < high ? z_sum : high;
    }
  }
  low = low < one ? one : low;
  high = high < low ? low : high;
  if (set.least > 1.f)
    low = high = one;
  ask(locate(set.below(low) + 1), locate(set.below(high) + 1));
  if (l == 0) {
    d.f.all = all, d.f.by_k = by_k, d.f.least_from = least_from, d.f.least_to = least_to;
    d.kept[0] = d.kept[1] = all; // (until a word says less; and what lies in front of min_p's buckets)
    d.kept[2] = least_from < kBuckets ? locate.start_of(least_from) : all;
    // (below the last bucket's end, for all roundings)
    const double end = set.most - (lowest + 2) * 2.0 / (double)buckets.by;
    d.f.floor = buckets.by > 0.f ? (float)(end - 1e-6 * (fabs(end) + fabs(set.most))) : -INFINITY;
  }
}

// The words of those buckets, to the list.
template <int NT, int DT>
__device__ __forceinline__ void gather(const SampleArgs &g, int64_t row, int from, int to, const Buckets &buckets, Draw<NT> &d) {
  using W = Words<DT>;
  const float floor = d.f.floor;
  for_words<NT, DT, NT == 64 ? 2 : 4>(g, row, from, to, [&](const float(&v)[W::N], int i) {
    uint32_t hits = 0;
    float top = v[0];
#pragma unroll
    for (int e = 1; e < W::N; ++e)
      top = fmaxf(top, v[e]);
    if (!(top >= floor)) // (most, where few words weigh much)
      return;
#pragma unroll
    for (int e = 0; e < W::N; ++e) {
      const int b = buckets.of(v[e]);
      hits |= (d.asked[b >> 5] >> (b & 31) & 1) << e;
    }
    if (hits) { // (few)
#pragma unroll
      for (int e = 0; e < W::N; ++e)
        if (hits >> e & 1) {
          const int at = atomicAdd(&d.filled, 1);
          if (at < list_of(NT))
            d.logits[at] = v[e], d.places[at] = (uint32_t)(i + e);
        }
    }
  });
  __syncthreads();
}

// The value of the lane whose number differs in one bit.
template <int FAR> __device__ __forceinline__ uint32_t other_lane(uint32_t v) {
  auto move = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 15, 15, false);
  };
  if constexpr (FAR == 1)
    return move(v, std::integral_constant<int, 0xB1>{}); // quad_perm [1,0,3,2]
  else if constexpr (FAR == 2)
    return move(v, std::integral_constant<int, 0x4E>{}); // quad_perm [2,3,0,1]
  else if constexpr (FAR == 4) // mirrored in halves of a row, then in quads
    return move(move(v, std::integral_constant<int, 0x141>{}), std::integral_constant<int, 0x1B>{});
  else if constexpr (FAR == 8)
    return move(v, std::integral_constant<int, 0x128>{}); // row_ror 8
  else {
    // odd rows (or the upper half) of one copy against even ones (the lower half) of another
    const auto both = FAR == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                                : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & FAR ? both[0] : both[1];
  }
}
// A word as one number, the larger the earlier in the order: key and index are 56 bits, and as many bits
// of a positive f64 below 2 compare as they do, at four times the rate of whole numbers of 64 bits.  0: none.
__device__ __forceinline__ double word_of(float logit, uint32_t place) {
  return __builtin_bit_cast(double, (uint64_t)key_of(logit) << 30 | (uint64_t)(~place & 0xFFFFFFu) << 6);
}
__device__ __forceinline__ float logit_of_word(double v) {
  return logit_of((uint32_t)(__builtin_bit_cast(uint64_t, v) >> 30));
}
__device__ __forceinline__ int32_t place_of_word(double v) {
  return (int32_t)(~(uint32_t)(__builtin_bit_cast(uint64_t, v) >> 6) & 0xFFFFFFu);
}
__device__ __forceinline__ void exchange(double &larger, double &smaller) {
  const double a = larger, b = smaller;
  const bool turned = b > a;
  larger = turned ? b : a, smaller = turned ? a : b;
}
template <int FAR> __device__ __forceinline__ void exchange_lanes(double (&v)[kOwn]) {
#pragma unroll
  for (int h = 0; h < kOwn; ++h) {
    const uint64_t own = __builtin_bit_cast(uint64_t, v[h]);
    const double w = __builtin_bit_cast(double, (uint64_t)other_lane<FAR>((uint32_t)(own >> 32)) << 32 | other_lane<FAR>((uint32_t)own));
    v[h] = (w > v[h]) == ((threadIdx.x & FAR) == 0) ? w : v[h];
  }
}

// n words in descending order, words kOwn * thread + h in a thread (0 behind the last): a bitonic network.
// Where a block is to ascend its words change their sign meanwhile.  Exchanges at distances below
// kOwn inside a thread, below 64 kOwn by DPP inside a wavefront, others through LDS (two places in turn: one
// barrier each); wavefronts in whose block nothing lies only keep the barriers.
template <int NT> __device__ __forceinline__ void sort_words(double (&v)[kOwn], int n, double (*swap)[NT * kOwn]) {
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t & ~63);
  exchange(v[0], v[1]);
  exchange(v[3], v[2]);
  uint32_t signs = 0;
  auto ascend = [&](uint32_t now) {
#pragma unroll
    for (int h = 0; h < kOwn; ++h)
      v[h] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, v[h]) ^ (uint64_t)(signs ^ now) << 32);
    signs = now;
  };
  int turn = 0;
#pragma clang loop unroll(disable)
  for (int size = 4; size < 2 * n; size *= 2) {
    const bool used = (wave * kOwn & -size) < n;
    if (used)
      ascend((t * kOwn & size) != 0 ? 0x80000000u : 0u);
#pragma clang loop unroll(disable)
    for (int far = size / 2; far >= 64 * kOwn; far /= 2) {
      if (used)
#pragma unroll
        for (int h = 0; h < kOwn; ++h)
          swap[turn][h * NT + t] = v[h];
      __syncthreads();
      if (used)
#pragma unroll
        for (int h = 0; h < kOwn; ++h) {
          const double w = swap[turn][h * NT + (t ^ far / kOwn)];
          v[h] = (w > v[h]) == ((t * kOwn & far) == 0) ? w : v[h];
        }
      turn ^= 1;
    }
    if (used) {
      if (size > 32 * kOwn)
        exchange_lanes<32>(v);
      if (size > 16 * kOwn)
        exchange_lanes<16>(v);
      if (size > 8 * kOwn)
        exchange_lanes<8>(v);
      if (size > 4 * kOwn)
        exchange_lanes<4>(v);
      if (size > 2 * kOwn)
        exchange_lanes<2>(v);
      if (size > kOwn)
        exchange_lanes<1>(v);
      exchange(v[0], v[2]);
      exchange(v[1], v[3]);
      exchange(v[0], v[1]);
      exchange(v[2], v[3]);
    }
  }
  ascend(0);
}

// The same of at most NT words, one in a thread (to swap[1]): a word's place is how many are larger.  Shorter code
// than the network's, which is what counts where few words make code run once.
template <int NT, int ROOM> __device__ __forceinline__ void rank_words(double v, int n, double (*swap)[ROOM]) {
  typedef double Two __attribute__((ext_vector_type(2)));
  constexpr int STEP = 8;
  const int t = threadIdx.x;
  swap[0][t] = v; // (zeros behind the last)
  __syncthreads();
  if (__builtin_amdgcn_readfirstlane(t & ~63) < n) {
    int larger = 0;
    for (int i = 0; i < n; i += STEP)
#pragma unroll
      for (int e = 0; e < STEP; e += 2) {
        const Two w = *(const Two *)&swap[0][i + e];
        larger += w[0] > v;
        larger += w[1] > v;
      }
    if (t < n)
      swap[1][larger] = v;
  }
  __syncthreads();
}

// The token of a row, from words that registers hold: in order, with their sums next to them, they answer
// every question by a comparison.  (A search for each of them in the list takes three times as long.)
template <int NT>
__device__ __forceinline__ void answer_sorted(const SampleArgs &g, int64_t row, const Settings &set, const Buckets &buckets,
                                              int n, Draw<NT> &d) {
  const int t = threadIdx.x, l = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  double v[kOwn];
  if (n <= kRanked && n <= NT) {
    const double own = t < n ? word_of(d.logits[t], d.places[t]) : 0.0;
    __syncthreads(); // (the words to sort lie where the list does)
    rank_words<NT>(own, n, d.swap);
#pragma unroll
    for (int h = 0; h < kOwn; ++h)
      v[h] = t * kOwn + h < n ? d.swap[1][t * kOwn + h] : 0.0;
  } else {
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      const int i = t * kOwn + h;
      v[h] = i < n ? word_of(d.logits[i], d.places[i]) : 0.0;
    }
    __syncthreads();
    sort_words<NT>(v, n, d.swap);
  }
  // sums up to each word of the list, then of the row: a bucket's begin at its first word
  const bool used = wave * 64 * kOwn < n;
  uint64_t weight[kOwn], up_to[kOwn], sum = 0;
  float x[kOwn];
  int home[kOwn];
  __syncthreads();
  if (used) {
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      const bool mine = v[h] > 0.0;
      x[h] = logit_of_word(v[h]);
      weight[h] = mine ? set.held(x[h]) : 0;
      home[h] = mine ? buckets.of(x[h]) : kBuckets;
      up_to[h] = sum += weight[h];
    }
    sum = sum_up_to_lane(sum);
    if (l == 63)
      d.bins.sum[wave] = sum;
    d.swap[0][t] = home[kOwn - 1];
  }
  __syncthreads();
  if (used) {
    sum -= up_to[kOwn - 1];
    for (int w = 0; w < wave; ++w)
      sum += d.bins.sum[w];
#pragma unroll
    for (int h = 0; h < kOwn; ++h) {
      up_to[h] += sum;
      const int before = h > 0 ? home[h > 0 ? h - 1 : 0] : t > 0 ? (int)d.swap[0][t - 1] : -1;
      if (home[h] < kBuckets && before != home[h]) {
        d.f.before[bucket_place(home[h])] -= up_to[h] - weight[h]; // (unsigned: wraps and wraps back)
        d.f.first[bucket_place(home[h])] -= (uint32_t)(t * kOwn + h);
      }
    }
  }
  __syncthreads();
  const int least_from = d.f.least_from, least_to = d.f.least_to, by_k = d.f.by_k;
  // (those behind the last word end nothing: their weight is 0)
  auto each = [&](auto take) {
    if (used)
#pragma unroll
      for (int h = 0; h < kOwn; ++h)
        take(h);
  };
  each([&](int h) {
    if (home[h] == kBuckets)
      return;
    up_to[h] += d.f.before[bucket_place(home[h])];
    const uint32_t rank = d.f.first[bucket_place(home[h])] + (uint32_t)(t * kOwn + h);
    if (by_k >= 0 && rank + 1 == (uint32_t)set.k)
      d.kept[0] = up_to[h];
  });
  // whoever ends a prefix says so
  auto ends = [&](int h, uint64_t need) { return up_to[h] - weight[h] < need && need <= up_to[h]; };
  uint64_t kept = d.f.all;
  if (by_k >= 0) {
    __syncthreads();
    kept = d.kept[0];
  }
  if (set.p < 1.f) {
    const uint64_t need = set.share(kept);
    each([&](int h) {
      if (ends(h, need))
        d.kept[1] = up_to[h];
    });
    __syncthreads();
    kept = d.kept[1] < kept ? d.kept[1] : kept;
  }
  if (set.least > 0.f && least_from < kBuckets) {
    // (the largest sum among them, or what lies in front of their buckets)
    uint64_t most = 0;
    each([&](int h) {
      if (home[h] >= least_from && home[h] <= least_to && set.weight(x[h]) >= least_bound(set))
        most = up_to[h];
    });
    if (used) {
      most = largest_of_wave<uint64_t>(most);
      if (l == 0 && most)
        atomicMax((unsigned long long *)&d.kept[2], (unsigned long long)most);
    }
    __syncthreads();
    kept = d.kept[2] < kept ? d.kept[2] : kept;
  }
  if (set.least > 1.f)
    kept = (uint64_t)1 << set.bits;
  const uint64_t need = set.below(kept) + 1;
  each([&](int h) {
    if (ends(h, need)) {
      g.token[row] = place_of_word(v[h]);
      if (g.probability)
        g.probability[row] = (float)((double)weight[h] / (double)kept);
    }
  });
}

// The token of a row, from the n words of the list; `handed` holds those that LDS does not.
template <int NT>
__device__ __forceinline__ void answer(const SampleArgs &g, int64_t row, const Settings &set, const Buckets &buckets, int n,
                                       Draw<NT> &d, const unsigned long long *handed = nullptr) {
  const int l = threadIdx.x & 63;
  // (Many equal logits, many that are close below one far above them, or distinct ones of a million words and more, of
  // which a bucket holds thousands: f32 2^20 normal ones 33 to 60 us, 2^22 94 us on the list and 29 to 46 ms here.)
  if (n > (handed ? kList : list_of(NT))) {
    sample_row<NT>(g, row, d.whole);
    return;
  }
  if (n <= sorted_of(NT)) {
    answer_sorted<NT>(g, row, set, buckets, n, d);
    return;
  }
  auto of_memory = [&](int i) { return __hip_atomic_load(&handed[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto logit_at = [&](int i) {
    return !handed || i < list_of(NT) ? d.logits[i] : __builtin_bit_cast(float, (uint32_t)of_memory(i));
  };
  auto place_at = [&](int i) { return !handed || i < list_of(NT) ? d.places[i] : (uint32_t)(of_memory(i) >> 32); };
  const uint64_t one = (uint64_t)1 << set.bits;
  const uint64_t all = d.f.all;
  const Locator locate{d.f, d.f.before[l * 17], l < 63 ? d.f.before[l * 17 + 17] : all};
  const int by_k = d.f.by_k, least_from = d.f.least_from, least_to = d.f.least_to;
  const bool by_p = set.p < 1.f;
  // The questions in turn: what the first k weigh, how far top_p reaches, which word is drawn, and its
  // index among those that are equal.  (One loop, so that the search is in the code once.)
  uint64_t kept = all;
  float word = 0.f;
  uint32_t drawn = 0;
  for (int q = by_k >= 0 ? 0 : by_p ? 1 : 2;; q = q == 0 && !by_p ? 2 : q + 1) {
    uint64_t need = drawn;
    int home = by_k;
    if (q == 0) {
      need = (uint64_t)set.k - d.f.first[bucket_place(home)];
    } else if (q < 3) {
      if (q == 2 && set.least > 0.f && least_from < kBuckets) {
        const double bound = least_bound(set);
        uint64_t large = 0;
        for (int i = threadIdx.x; i < n; i += NT) {
          const float x = logit_at(i);
          const int at = buckets.of(x);
          if (at >= least_from && at <= least_to && set.weight(x) >= bound)
            large += set.held(x);
        }
        if (threadIdx.x == 0)
          d.bins.sum[0] = 0;
        __syncthreads();
        large = of_lane(sum_up_to_lane(large), 63);
        if (l == 0 && large)
          atomicAdd((unsigned long long *)&d.bins.sum[0], (unsigned long long)large);
        __syncthreads();
        large = locate.start_of(least_from) + d.bins.sum[0];
        kept = large < kept ? large : kept;
        __syncthreads();
      }
      if (q == 2 && set.least > 1.f)
        kept = one;
      need = q == 1 ? set.share(kept) : set.below(kept) + 1;
      home = locate(need);
      need -= locate.start_of(home);
    }
    const bool by_place = q == 3;
    const End e = list_end<NT>(
        q == 0 || by_place, need, n, d,
        [&](int i) {
          const float x = logit_at(i);
          return by_place ? (x == word ? ~place_at(i) : 0u) : buckets.of(x) == home ? key_of(x) : 0u;
        },
        [&](uint32_t key) { return by_place ? 0ull : set.held(logit_of(key)); });
    if (q < 2) {
      kept = locate.start_of(home) + e.sum + e.ties * set.held(logit_of(e.key));
    } else if (q == 2) {
      drawn = e.ties;
      word = logit_of(e.key);
      if (threadIdx.x == 0 && g.probability)
        g.probability[row] = (float)((double)set.held(word) / (double)kept);
      if (e.same == 1) { // (its only place)
        for (int i = threadIdx.x; i < n; i += NT)
          if (logit_at(i) == word)
            g.token[row] = (int32_t)place_at(i);
        return;
      }
    } else {
      if (threadIdx.x == 0)
        g.token[row] = (int32_t)~e.key;
      return;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ bool counts_words(const SampleArgs &g, int k) { return k > 0 && k < g.words; }

// A workgroup a row.
template <int NT, int DT> __global__ __launch_bounds__(NT) void sample_whole_kernel(SampleArgs g) {
  __shared__ Draw<NT> d;
  __shared__ Sums sums;
  __shared__ RangeRoom<NT> room;
  const int64_t row = blockIdx.x;
  const Asked asked(g, row);
  const Range range = range_of<NT, DT>(g, row, 0, g.words, room);
  if (settled<NT>(g, row, range, asked.t, d.whole))
    return;
  const Settings set(g, asked, range.largest());
  const Buckets buckets(set, range.least);
  const bool count = counts_words(g, set.k);
  sums_of<NT, DT>(g, row, 0, g.words, set, buckets, count, sums);
  if (threadIdx.x < 64) {
    Sixteen own;
    own.load(&sums.sum[threadIdx.x * 17], &sums.count[threadIdx.x * 17]);
    ask_buckets<NT>(set, buckets, count, own, d);
  }
  __syncthreads();
  gather<NT, DT>(g, row, 0, g.words, buckets, d);
  answer<NT>(g, row, set, buckets, d.filled, d);
}

template <int DT> __global__ __launch_bounds__(kThreads) void sample_most_kernel(SampleArgs g) {
  __shared__ RangeRoom<kThreads> room;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  if (part == 0) {
    g.sums[row * kBuckets + threadIdx.x] = 0, g.counts[row * kBuckets + threadIdx.x] = 0;
    if (threadIdx.x == 0)
      g.filled[row] = 0, g.arrived[row] = 0;
  }
  const int from = part * g.part_words, to = from + g.part_words < g.words ? from + g.part_words : g.words;
  const Range r = range_of<kThreads, DT>(g, row, from, to, room);
  if (threadIdx.x == 0) {
    g.part_most[row * g.parts + part] = r.most;
    g.part_least[row * g.parts + part] = r.least;
  }
}

// (a lane a part, at most 32)
__device__ __forceinline__ Range range_of_parts(const SampleArgs &g, int64_t row) {
  const int p = threadIdx.x & 31, at = p < g.parts ? p : 0;
  Range r;
  r.most = largest_of_wave<uint64_t>(g.part_most[row * g.parts + at]);
  r.least = logit_of(~largest_of_wave<uint32_t>(~key_of(g.part_least[row * g.parts + at])));
  return r;
}

template <int DT> __global__ __launch_bounds__(kThreads) void sample_sums_kernel(SampleArgs g) {
  __shared__ Sums sums;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  const Asked asked(g, row);
  const Range range = range_of_parts(g, row);
  if (!has_questions(range, asked.t))
    return;
  const Settings set(g, asked, range.largest());
  const Buckets buckets(set, range.least);
  const bool count = counts_words(g, set.k);
  const int from = part * g.part_words, to = from + g.part_words < g.words ? from + g.part_words : g.words;
  sums_of<kThreads, DT>(g, row, from, to, set, buckets, count, sums);
  const int at = bucket_place((int)threadIdx.x);
  if (sums.sum[at])
    atomicAdd(&g.sums[row * kBuckets + threadIdx.x], sums.sum[at]);
  if (count && sums.count[at])
    atomicAdd(&g.counts[row * kBuckets + threadIdx.x], sums.count[at]);
}

// A workgroup a part: all find the buckets in question for themselves and bring the words of their part
// together; the last one to have written them answers.
//
// What they hand over goes through atomics of device scope, which are coherent over the chip by
// themselves: every thread waits for its stores, then the workgroup adds itself to those that have
// arrived.  (Fences would write back and discard the L2 caches: 165 us for 48 rows, all in all.)
template <int DT> __global__ __launch_bounds__(kDraw, 4) void sample_draw_kernel(SampleArgs g) {
  __shared__ Draw<kDraw> d;
  __shared__ uint32_t told;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  const Asked asked(g, row);
  Sixteen own;
  if (threadIdx.x < 64)
    own.load(g.sums + row * kBuckets + threadIdx.x * 16, g.counts + row * kBuckets + threadIdx.x * 16);
  const Range range = range_of_parts(g, row);
  if (!has_questions(range, asked.t)) {
    if (part == 0)
      settled<kDraw>(g, row, range, asked.t, d.whole);
    return;
  }
  const Settings set(g, asked, range.largest());
  const Buckets buckets(set, range.least);
  if (threadIdx.x < 64)
    ask_buckets<kDraw>(set, buckets, counts_words(g, asked.k), own, d);
  __syncthreads();
  const int from = part * g.part_words, to = from + g.part_words < g.words ? from + g.part_words : g.words;
  gather<kDraw, DT>(g, row, from, to, buckets, d);
  constexpr uint32_t HERE = list_of(kDraw);
  unsigned long long *const list = g.list + row * kList;
  const uint32_t mine = (uint32_t)d.filled;
  if (threadIdx.x == 0)
    told = mine ? __hip_atomic_fetch_add(&g.filled[row], mine > HERE ? kList + 1 : mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
  __syncthreads();
  const uint32_t first = told;
  for (uint32_t i = threadIdx.x; i < mine && i < HERE && first + i < kList; i += kDraw)
    __hip_atomic_store(&list[first + i],
                       (unsigned long long)d.places[i] << 32 | __builtin_bit_cast(uint32_t, d.logits[i]), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup"); // (for the compiler)
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0)
    told = __hip_atomic_fetch_add(&g.arrived[row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (told != (uint32_t)g.parts - 1)
    return;
  const uint32_t n = __hip_atomic_load(&g.filled[row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (uint32_t i = threadIdx.x; i < n && i < HERE; i += kDraw) {
    const unsigned long long v = __hip_atomic_load(&list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    d.logits[i] = __builtin_bit_cast(float, (uint32_t)v), d.places[i] = (uint32_t)(v >> 32);
  }
  __syncthreads();
  answer<kDraw>(g, row, set, buckets, (int)n, d, list);
}

// How rows are cut: a workgroup a row where rows are short or fill the chip, otherwise parts that do, of
// 4096 words at least.  us, one part / parts: bf16 33 x 16384 17.2 / 20.9 (four), f32 4 x 8192 13.7 / 17.9;
// f32 130 x 131072 80 / 67 (four), 256 x 131072 94 / 108 (two), bf16 257 x 32000 31 / 40.  As it is, over
// 131072 words f32 (128256 words bf16): 128 rows 65 us (59), 191 92 (79), 192 82 (74), 256 88 (76), 257 126 (77),
// 300 138 (116), 512 163 (144): a workgroup of 1024 threads has a compute unit to itself, and more of them than units
// take a second round.
constexpr int64_t kFull = 192, kShort = 20480;
struct Cut {
  int parts, words;
  Cut(int64_t rows, int64_t row_words) {
    int64_t n = rows >= kFull || row_words <= kShort ? 1 : (512 + rows - 1) / rows;
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

// (a grid's threads are a number below 2^32)
static bool side_by_side(const fhip_sample_desc &d) {
  return (d.logits.stride[1] == 1 || d.logits.dim[1] == 1) && d.logits.dim[0] < (1 << 21);
}
// Where things lie in the workspace, which begins with the parts' largest logits.
struct Places {
  size_t least, sums, counts, filled, list, bytes;
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
  p.counts = p.sums + (size_t)d.logits.dim[0] * kBuckets * 8;
  p.filled = p.counts + (size_t)d.logits.dim[0] * kBuckets * 4;
  p.list = p.filled + up((size_t)d.logits.dim[0] * 8);
  p.bytes = p.list + (size_t)d.logits.dim[0] * kList * 8;
  return p;
}

template <int DT> static int launch(fhip_ctx *ctx, const SampleArgs &g) {
  if (g.parts == 1) {
    const dim3 grid((unsigned)g.rows);
    if (g.words <= 1024)
      hipLaunchKernelGGL((sample_whole_kernel<64, DT>), grid, dim3(64), 0, ctx->stream, g);
    else if (g.words <= 8192)
      hipLaunchKernelGGL((sample_whole_kernel<256, DT>), grid, dim3(256), 0, ctx->stream, g);
    else
      hipLaunchKernelGGL((sample_whole_kernel<1024, DT>), grid, dim3(1024), 0, ctx->stream, g);
  } else { // (fewer than kFull rows)
    const dim3 grid((unsigned)g.parts, (unsigned)g.rows);
    hipLaunchKernelGGL(sample_most_kernel<DT>, grid, dim3(kThreads), 0, ctx->stream, g);
    hipLaunchKernelGGL(sample_sums_kernel<DT>, grid, dim3(kThreads), 0, ctx->stream, g);
    hipLaunchKernelGGL(sample_draw_kernel<DT>, grid, dim3(kDraw), 0, ctx->stream, g);
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
  if (side_by_side(*d)) {
    const Cut c(g.rows, g.words);
    g.parts = c.parts, g.part_words = c.words;
    char *w = (char *)workspace;
    g.part_most = (uint64_t *)w, g.part_least = (float *)(w + at.least);
    g.sums = (unsigned long long *)(w + at.sums), g.counts = (uint32_t *)(w + at.counts);
    g.filled = (uint32_t *)(w + at.filled), g.arrived = g.filled + g.rows, g.list = (unsigned long long *)(w + at.list);
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
