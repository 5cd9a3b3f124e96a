// Attention of each sequence's newest rows over its keys in a paged cache, on
// MFMA: bf16 / f16, head dim 64 or 128, pages of a multiple of 16 rows, the
// cache in the rows' type or in 4 bits.
//
// Bound by reading each sequence's keys and values once.  The rows that share a
// key / value head -- positions times grouped heads -- are packed into tiles of
// 16, position after position; a wavefront walks chunks of 32 keys as in
// sdpa_decode.hip:
//   * S^T = K Q^T on 16 x 16 x 32 MFMAs, K fragments straight from the pages; a
//     lane ends up with 8 keys of one row;
//   * online softmax in those lanes; the rounded probabilities are the operand
//     of the next product as they lie;
//   * O^T += V^T P^T, from 8 rows of V per lane.
// A chunk's two tiles of 16 keys lie in one page each.  A wavefront looks the
// pages of its next 32 chunks up with one load, one tile per lane, and takes
// them from there as scalars: no load waits for a page number.
//
// 4 bits: a value is low + scale c with c in 0 .. 15, so for each group
//   Q . K = scale (Q . c) + low (sum of Q),   P V = (P scale) c + (P . low):
// the codes go into the products as they are, 3 bits' worth of work away from
// the type's own numbers (a nibble below the exponent of 128 in bf16, of 1024 in f16
// is 128 + c or 1024 + c exactly; K's offset is in the accumulator's start or
// taken off, V's comes from a product with ones), scales and lows act on sums and
// probabilities in f32.  P scale is rounded where P would be; so that its rounding
// meets no larger numbers than in 16 bits, the codes count from the middle, as
// c - 8, and 8 (P . scale) goes with the lows; in the end the codes' part is scaled
// by the sum of P scale over that of its rounded values.  Each product's 32 dims (K) or 16 columns (V) lie within a group.
//
// In 4 bits a chunk is 4 KB, and more of them have to be on their way: rows and parameters go
// to a ring of stages in the wavefront's own LDS by LDS-DMA, from which each lane takes
// what its fragments need.
//
// Work: no one but the device knows the lengths.  All sequences' chunks, one
// tile and head after another, are one line that is cut into pieces, one per
// workgroup; each finds its own from the lengths.  What a workgroup does of
// a (sequence, tile, head) is a segment: whole ones it stores, parts meet in the
// workspace, in a fixed order, in a second kernel.  A cut near a segment's end moves
// there: a new segment waits for its first loads, 3 us in which its workgroup reads nothing.
// Where the page table has room for few keys only, or there are many tiles, a workgroup
// takes one whole (sequence, tile, head).
//
// bf16, 32 heads on 8 of 128: one token of each of 32 sequences of 16 to 8192 keys (354 MB) 66.9 us, 5.3 TB/s; of 64 with
// 8192 keys each 320 us, 6.7 TB/s, a reading stream's rate.  4 bits, groups of 64: three tokens of 64 sequences of 16 to 16384
// keys (391 MB) 91.5 us, 4.3 TB/s, one of 64 with 8192 124 us, 4.9 TB/s: the vector ALU works 71 % of the time on codes, scales
// and probabilities (309 instructions a chunk), for two wavefronts a SIMD about what it can.
#include "paged_cache.h"
#include "fast_paths.h"

#include <cmath>
#include <type_traits>

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
#define PG_AS1 __attribute__((address_space(1)))
#define PG_AS3 __attribute__((address_space(3)))

constexpr int kWaves = 4;
constexpr int kChunk = 32; // keys of a step
constexpr float kNegBig = -1.0e30f;

struct PagedArgs {
  const char *q;
  char *o;
  int64_t q_st, q_sh, o_st, o_sh; // row and head strides in elements
  const int32_t *offsets;
  FhipCacheView cache;
  int32_t T, Hkv, group; // group: query heads per key head
  int32_t causal;
  int32_t pieces; // workgroups that share the line
  int32_t *upto;  // of many sequences, their work summed up to each (null: few)
  float scale_log2e;
  // of sequences in several pieces (null: there are none)
  struct Info {
    int32_t first; // the sequence's place on the line
    int32_t chunks, pos, tiles;
    int32_t large, small; // chunks of the pieces
  } *info;        // [T]
  float *part;    // [piece][2][16][HD] sums: of a segment that another piece began, and of one that it goes on with
  float *part_ml; // [piece][2][16] (m, l)
};

// Keys up to which no sequence is cut (the launch that joins pieces takes longer than what it saves).
constexpr int64_t kWhole = 1024;

template <bool BF16>
__device__ __forceinline__ f32x4 pg_mfma(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF16> __device__ __forceinline__ uint32_t pg_pack(float a, float b) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
  } else {
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  }
}

template <bool BF16> __device__ __forceinline__ float pg_value(uint32_t pair, int i) {
  if constexpr (BF16)
    return __builtin_bit_cast(float, i ? pair & 0xffff0000u : pair << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i ? pair >> 16 : pair));
}

template <bool BF16> __device__ __forceinline__ void pg_store(char *o, int64_t at, float v) {
  if constexpr (BF16)
    ((PG_AS1 __bf16 *)o)[at] = (__bf16)v;
  else
    ((PG_AS1 _Float16 *)o)[at] = (_Float16)v;
}

// Nibbles i and i + 4 of a word as two 16-bit numbers, both `kOffset` too large.  (The masks are
// hidden from the compiler, which would otherwise take two instructions for what v_and_or_b32
// does with one scalar and one vector operand.)
template <bool BF16> struct Codes {
  static constexpr float kOffset = BF16 ? 128.f : 1024.f;
  uint32_t mask = 0x000f000fu, exponent = BF16 ? 0x43004300u : 0x64006400u;
  __device__ __forceinline__ Codes() { asm("" : "+s"(mask), "+v"(exponent)); }
  __device__ __forceinline__ uint32_t pair(uint32_t w, int i) const { return ((w >> (4 * i)) & mask) | exponent; }
};

// LDS reads that the compiler does not see as memory accesses (it would make each wait for every
// LDS-DMA in flight), and the wait that goes with them.
template <int OFFSET> __device__ __forceinline__ void pg_read(u32x4 &to, uint32_t from) {
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(to) : "v"(from), "n"(OFFSET));
}
template <int OFFSET> __device__ __forceinline__ void pg_read(u32x2 &to, uint32_t from) {
  asm volatile("ds_read_b64 %0, %1 offset:%2" : "=v"(to) : "v"(from), "n"(OFFSET));
}
template <int OFFSET> __device__ __forceinline__ void pg_read(uint32_t &to, uint32_t from) {
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(to) : "v"(from), "n"(OFFSET));
}
template <int OFFSET> __device__ __forceinline__ void pg_read16(uint32_t &to, uint32_t from) {
  asm volatile("ds_read_u16 %0, %1 offset:%2" : "=v"(to) : "v"(from), "n"(OFFSET));
}
template <int OFFSET> __device__ __forceinline__ void pg_read8(uint32_t &to, uint32_t from) {
  asm volatile("ds_read_u8 %0, %1 offset:%2" : "=v"(to) : "v"(from), "n"(OFFSET));
}
__device__ __forceinline__ void pg_lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// (behind the wait: nothing that uses `x` moves in front of it)
template <typename V> __device__ __forceinline__ void pg_pin(V &x) { asm volatile("" : "+v"(x)); }

template <int N, typename F> __device__ __forceinline__ void pg_static_for(F &&f) {
  if constexpr (N > 0) {
    pg_static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// 16 or 4 bytes per lane from memory to LDS, lane after lane from `to`.  (The builtin takes its size as
// a literal, and 16 only for this device.)
// ONCE: what nothing reads again (non-temporal).
#if defined(__HIP_DEVICE_COMPILE__)
#define PG_DMA(BYTES)                                                                            \
  __builtin_amdgcn_global_load_lds((const PG_AS1 void *)from,                                    \
                                   (PG_AS3 void *)(uintptr_t)__builtin_amdgcn_readfirstlane(to), \
                                   BYTES, 0, ONCE ? 2 : 0)
#else
#define PG_DMA(BYTES)
#endif
template <bool ONCE> __device__ __forceinline__ void pg_dma16(const char *from, uint32_t to) { PG_DMA(16); }
template <bool ONCE> __device__ __forceinline__ void pg_dma4(const char *from, uint32_t to) { PG_DMA(4); }
template <bool ONCE, typename V> __device__ __forceinline__ V pg_load(const char *from) {
  const PG_AS1 V *p = (const PG_AS1 V *)from;
  return ONCE ? __builtin_nontemporal_load(p) : *p;
}

// s_waitcnt vmcnt(vm) alone.
__device__ __forceinline__ constexpr int pg_wait_imm(int vm) {
  return (vm & 0xF) | ((vm >> 4) << 14) | (0x7 << 4) | (0xF << 8);
}

// Bytes of LDS per wavefront: its sums in the end (17 floats per column of O); in 4 bits before that a ring of stages,
// each 32 rows of K, of V and their (scale, low) pairs.
template <int HD, int G> struct PagedShape {
  static constexpr bool kQ4 = G != 0;
  static constexpr int kGroups = HD / (kQ4 ? G : HD);
  static constexpr int kRow = HD / 2; // bytes of a row in 4 bits
  static constexpr int kPairs = 64 * kRow;
  static constexpr int kStage = kPairs + 256 * kGroups;
  static constexpr int kStages = kGroups == 4 ? 3 : 4; // (two workgroups' in 160 KB)
  static constexpr int kSums = HD * 17 * 4;
  static constexpr int kBytes = kQ4 && kStages * kStage > kSums ? kStages * kStage : kSums;
};

// Inclusive sums over the wavefront's lanes.
template <typename V> __device__ __forceinline__ V pg_scan(V x) {
  auto add = [&](auto ctrl, auto rows) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                              decltype(rows)::value, 0xf, false);
    x += __builtin_bit_cast(V, y);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}); // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}); // row_bcast 15, 31
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return x;
}
template <typename V> __device__ __forceinline__ V pg_lane(V x, int lane) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

// A sequence as the split sees it.
struct Sequence {
  int start, rows;  // packed rows
  int length;       // keys
  int tiles, chunks;
};
__device__ __forceinline__ Sequence pg_sequence(const PagedArgs &g, int b) {
  Sequence s;
  const FhipRows r = fhip_rows_between(g.offsets[b], g.offsets[b + 1], g.T);
  s.start = r.first, s.rows = r.count;
  const int len = g.cache.lengths[b];
  s.length = len < 0 ? 0 : len;
  const int room = g.cache.table_pages * g.cache.page_size; // <= 2^30
  const int keys = s.length < room ? s.length : room;
  s.tiles = (int)(((int64_t)s.rows * g.group + 15) / 16);
  s.chunks = keys ? (keys + kChunk - 1) / kChunk : 1;
  return s;
}

// A sequence's part of the line: the chunks of its tiles and heads, or where none is cut those; fewer than 2^31 in all.
__device__ __forceinline__ int pg_work(const PagedArgs &g, const Sequence &s) {
  return s.tiles * g.Hkv * (g.info ? s.chunks : 1);
}

// More sequences than a wavefront has lanes: a first kernel sums their work up to each, and the workgroups search in that
// 64 at a time.  Walked over by each workgroup, 1024 of 500 keys took 464 us, like this 360; 64 25.5 and 27.4.
constexpr int kLanes = 64;
__global__ __launch_bounds__(1024) void sdpa_paged_index_kernel(PagedArgs g) {
  __shared__ int sums[16];
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int total = 0;
  for (int b0 = 0; b0 < g.cache.batch; b0 += 1024) {
    const int b = b0 + (int)threadIdx.x;
    const int x = pg_scan(b < g.cache.batch ? pg_work(g, pg_sequence(g, b)) : 0);
    if (l == 63)
      sums[wave] = x;
    __syncthreads();
    int front = total;
    for (int w = 0; w < 16; ++w) {
      front += w < wave ? sums[w] : 0;
      total += sums[w];
    }
    if (b < g.cache.batch)
      g.upto[b] = front + x;
    __syncthreads();
  }
}

// ONCE: rows share no keys but within a tile, as far as the host knows: a key is read once (non-temporal).
template <bool BF16, int HD, int G, bool ONCE>
__global__ __launch_bounds__(kWaves * 64)
__attribute__((amdgpu_waves_per_eu(2, 8))) void sdpa_paged_kernel(PagedArgs g) {
  constexpr bool Q4 = G != 0;
  constexpr int GG = Q4 ? G : HD;  // dims that share a scale
  constexpr int NG = HD / GG;      // groups
  constexpr int T = HD / 16;       // 16-column tiles of O
  constexpr int TG = GG / 16;      // of them per group; columns of a lane in it
  constexpr int KD = HD / 32;      // MFMA steps of a score tile
  constexpr int SG = GG / 32;      // of them per group
  constexpr int PITCH = 17;        // floats per column of O in LDS
  constexpr float kRedo = 8192.0f;
  // 4 bits under f16: P scale goes into the product, and scales are halves of any size.  So that it neither loses bits
  // below f16's normal numbers nor passes its largest, a row's probabilities carry a factor 2^lift, which begins (with
  // each new maximum) where the smallest half comes to 2^12, and falls to what brings the sum of a lane's products
  // below kMost.
  constexpr bool LIFT = Q4 && !BF16;
  constexpr int kLift = 36;
  constexpr float kMost = 32768.0f;
  using S = PagedShape<HD, G>;
  constexpr int ROW = S::kRow, SEGS = ROW / 16; // 4 bits: bytes of a row, 16-byte pieces of it
  constexpr int VB = GG / 32;      // bytes of a V row and group per lane
  static_assert(!Q4 || VB == 4 || VB == 2 || VB == 1, "groups of 32, 64 or 128");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float ml[kWaves][2][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = threadIdx.x & 63, lq = l & 15, lg = l >> 4;
  const FhipCacheView &c = g.cache;
  const Codes<BF16> codes;
  float *const sums = (float *)(smem + wave * S::kBytes);
  const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)(wave * S::kBytes);

  // ---- this workgroup's piece of the line ----------------------------------------
  const bool cut = g.info != nullptr;
  // Up to 64 sequences are kept for the segments' search, in LDS: registers are what limits the wavefronts.
  __shared__ Sequence front[64];
  __shared__ int front_upto[64];
  int total;
  if (g.upto) {
    total = g.upto[c.batch - 1];
  } else {
    const Sequence s = l < c.batch ? pg_sequence(g, l) : Sequence{};
    const int upto = pg_scan(pg_work(g, s));
    front_upto[l] = upto; // (every wavefront writes the same)
    front[l] = s;
    total = pg_lane(upto, 63);
  }
  int b = -1, first = 0; // a sequence and its place on the line
  Sequence seq{};
  auto find = [&](int at) { // the sequence that holds `at`
    if (g.upto) {
      b = fhip_first_above(g.upto, c.batch, at);
      if (b >= 0) {
        seq = pg_sequence(g, b);
        first = g.upto[b] - pg_work(g, seq);
      }
      return;
    }
    const Sequence s = front[l];
    const int upto = front_upto[l];
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > at);
    b = past ? __builtin_ctzll(past) : -1;
    if (past) {
      first = pg_lane(upto - pg_work(g, s), b);
      seq = Sequence{pg_lane(s.start, b), pg_lane(s.rows, b), pg_lane(s.length, b), pg_lane(s.tiles, b), pg_lane(s.chunks, b)};
    }
  };
  int at = (int)fhip_line_index(blockIdx.y), stop = at + 1;
  FhipPieces pieces{};
  if (cut) {
    pieces = FhipPieces::of(total, g.pieces);
    // the piece's ends, each at a segment's own where that is near
    const int64_t from = pieces.at(blockIdx.x);
    auto snapped = [&](int64_t x) {
      if (x >= total)
        return total;
      find((int)x);
      if (b < 0)
        return total;
      return pieces.moved((int)x, first, seq.chunks);
    };
    at = snapped(from);
    stop = snapped(pieces.at(blockIdx.x + 1));
  }
  if (at >= total)
    return;
  stop = stop < total ? stop : total;
  while (at < stop) {
    find(at);
    // (b < 0 and items behind the last: what offsets that overlap could lead to)
    const int unit = cut ? seq.chunks : 1;
    const int item = b < 0 ? 0 : (at - first) / unit;
    int c0 = at - first - item * unit;
    if (b < 0 || seq.tiles <= 0 || item < 0 || c0 < 0 || item / seq.tiles >= g.Hkv)
      return;
    int c1 = stop - at < unit - c0 ? c0 + stop - at : unit;
    at += c1 - c0;
    const bool whole = c0 == 0 && c1 == unit;
    const int slot = c0 == 0 ? 1 : 0;
    if (!cut)
      c1 = seq.chunks;
    // (tiles of a head side by side: they read the same keys)
    const int hk = item / seq.tiles, qt = item % seq.tiles;
    const int room = c.table_pages * c.page_size;
    const int keys = seq.length < room ? seq.length : room;
    const int left = seq.rows * g.group - qt * 16; // of the sequence's packed rows from this tile's first
    const int row = qt * 16 + (lq < left ? lq : left - 1);
    const int pos = row / g.group, hg = row - pos * g.group;
    // keys that this lane's row sees
    int seen = g.causal ? seq.length - seq.rows + pos + 1 : seq.length;
    const bool beyond = seen > keys; // of the page table
    seen = seen < 0 ? 0 : beyond ? keys : seen;
    int all_see = seen, any_sees = seen; // what every row sees: chunks up to it need no mask
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const int x = __shfl_xor(all_see, o, 64), y = __shfl_xor(any_sees, o, 64);
      all_see = x < all_see ? x : all_see;
      any_sees = y > any_sees ? y : any_sees;
    }
    all_see = __builtin_amdgcn_readfirstlane(all_see);
    if (cut && hk == 0 && slot == 1 && threadIdx.x < 16)
      g.info[seq.start + pos] = PagedArgs::Info{first, seq.chunks, pos, seq.tiles, pieces.large, pieces.small};
    // chunks behind the last key that any row sees have nothing
    const int need = (__builtin_amdgcn_readfirstlane(any_sees) + kChunk - 1) / kChunk;
    c1 = c1 < need ? c1 : need;
    const int steps = (c1 - c0 - wave + kWaves - 1) / kWaves; // this wavefront's chunks c0 + wave + 4 i

    // ---- Q fragments (B operand of S^T = K Q^T) ----------------------------------
    // step u of lane group lg: dims u * 32 + lg * 8 .. + 7; in 4 bits, step s of group n:
    // n * GG + lg * GG / 4 + s * 8 .. + 7, as a lane's codes of a group lie side by side
    uint32_t qf[KD][4];
    float qsum[NG]; // of this lane's row over a group's dims
    {
      const char *src = g.q + ((int64_t)(seq.start + pos) * g.q_st + (int64_t)(hk * g.group + hg) * g.q_sh) * 2;
#pragma unroll
      for (int u = 0; u < KD; ++u) {
        const int d = Q4 ? u / SG * GG + lg * (GG / 4) + u % SG * 8 : u * 32 + lg * 8;
        const u32x4 x = *(const PG_AS1 u32x4 *)(src + d * 2);
        if constexpr (Q4) { // the pairs that Codes::pair gives: (0, 4), (1, 5), (2, 6), (3, 7)
          qf[u][0] = __builtin_amdgcn_perm(x.z, x.x, 0x05040100u);
          qf[u][1] = __builtin_amdgcn_perm(x.z, x.x, 0x07060302u);
          qf[u][2] = __builtin_amdgcn_perm(x.w, x.y, 0x05040100u);
          qf[u][3] = __builtin_amdgcn_perm(x.w, x.y, 0x07060302u);
        } else {
          qf[u][0] = x.x, qf[u][1] = x.y, qf[u][2] = x.z, qf[u][3] = x.w;
        }
      }
    }

    // ---- loads -------------------------------------------------------------------
    constexpr int ES = Q4 ? 1 : 2; // bytes per stride unit
    const uint32_t k_slot = (uint32_t)(c.k.slot * ES), v_slot = (uint32_t)(c.v.slot * ES);
    const char *k_head = c.k.data + (int64_t)hk * c.k.head * ES;
    const char *v_head = c.v.data + (int64_t)hk * c.v.head * ES;
    const char *kp_head = (const char *)(c.k.params + (int64_t)hk * c.k.params_head);
    const char *vp_head = (const char *)(c.v.params + (int64_t)hk * c.v.params_head);
    // Of tile l & 1 of this wavefront's chunk (i & ~31) + (l >> 1): bytes to its first row in both pools and in
    // the parameters', and whether it has a page.
    struct Places {
      int64_t k, v, kp, vp;
      int bad;
    } places{};
    auto look_up = [&](int i) {
      const int key = ((c0 + wave + kWaves * (i + (l >> 1))) * 2 + (l & 1)) * 16;
      const uint32_t n = (uint32_t)key / (uint32_t)c.page_size;
      int page = 0, slot = 0;
      places.bad = 0;
      if (key < keys) { // (and so n < table_pages)
        slot = key - (int)n * c.page_size;
        page = c.table[b * c.table_stride + n];
        if ((uint32_t)page >= (uint32_t)c.pool_pages)
          page = 0, places.bad = 1;
      }
      places.k = ((int64_t)page * c.k.page + (int64_t)slot * c.k.slot) * ES;
      places.v = ((int64_t)page * c.v.page + (int64_t)slot * c.v.slot) * ES;
      if constexpr (Q4) {
        places.kp = ((int64_t)page * c.k.params_page + (int64_t)slot * c.k.params_slot) * 2;
        places.vp = ((int64_t)page * c.v.params_page + (int64_t)slot * c.v.params_slot) * 2;
      }
    };
    auto place = [&](int64_t x, int lane) {
      return ((int64_t)pg_lane((int)(x >> 32), lane) << 32) | (uint32_t)pg_lane((int)x, lane);
    };
    // LDS, 4 bits: piece s of row r lies at piece s ^ swizzle(r), which spreads the rows of one read over the banks.
    // LDS-DMA writes lane after lane: the lanes' own addresses are permuted.
    auto swizzle = [](int r) { return r / (256 / ROW) & (SEGS - 1); };
    // a lane's offsets from its tile's first row: 16 bits, its fragments; 4 bits, a piece of row l / SEGS (head dim 64: one
    // load for both tiles)
    const int piece = Q4 ? (l % SEGS ^ swizzle(l / SEGS)) * 16 : 0;
    const uint32_t k_lane = Q4 ? (uint32_t)(l / SEGS % 16) * k_slot + (uint32_t)piece : (uint32_t)lq * k_slot + (uint32_t)(lg * 16);
    const uint32_t v_lane = Q4 ? (uint32_t)(l / SEGS % 16) * v_slot + (uint32_t)piece : (uint32_t)(lg * 4) * v_slot + (uint32_t)(lq * T * 2);
    // .. and a pair of row l % (16 NG) / NG of a tile: 16 lanes (of K, then V, both tiles) per load and group
    const uint32_t pair_row = (uint32_t)(l % (16 * NG) / NG), pair_at = (uint32_t)(l % NG * 4);
    const uint32_t kp_lane = pair_row * (uint32_t)(c.k.params_slot * 2) + pair_at;
    const uint32_t vp_lane = pair_row * (uint32_t)(c.v.params_slot * 2) + pair_at;
    struct Chunk { // 16 bits
      u32x4 k[2 * KD], v[8];
      int bad;
    };
    auto fetch = [&](Chunk &x, int i) {
      if ((i & 31) == 0)
        look_up(i);
      const int lane = (i & 31) * 2;
      x.bad = pg_lane(places.bad, lane) | pg_lane(places.bad, lane + 1) << 1;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char *kt = k_head + place(places.k, lane + t), *vt = v_head + place(places.v, lane + t);
#pragma unroll
        for (int u = 0; u < KD; ++u)
          x.k[t * KD + u] = pg_load<ONCE, u32x4>(kt + u * 64 + k_lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char *p = vt + (uint64_t)r * v_slot + v_lane;
          if constexpr (T == 8) {
            x.v[t * 4 + r] = pg_load<ONCE, u32x4>(p);
          } else {
            const u32x2 y = pg_load<ONCE, u32x2>(p);
            x.v[t * 4 + r].x = y.x, x.v[t * 4 + r].y = y.y;
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int kDmas = SEGS + (NG == 4 ? 4 : NG); // 4 bits: LDS-DMA instructions of a chunk
    uint32_t bads = 0; // of the last 16 chunks issued, the newest lowest
    auto issue = [&](int i) { // chunk i, on its way to stage i % kStages
      if constexpr (Q4) {
        if ((i & 31) == 0)
          look_up(i);
        const int lane = (i & 31) * 2;
        bads = bads << 2 | (uint32_t)(pg_lane(places.bad, lane) | pg_lane(places.bad, lane + 1) << 1);
        const uint32_t stage = lds + (uint32_t)(i % S::kStages * S::kStage);
        const char *kt[2], *vt[2], *kpt[2], *vpt[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          kt[t] = k_head + place(places.k, lane + t);
          vt[t] = v_head + place(places.v, lane + t);
          kpt[t] = kp_head + place(places.kp, lane + t);
          vpt[t] = vp_head + place(places.vp, lane + t);
        }
        if constexpr (SEGS == 4) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            pg_dma16<ONCE>(kt[t] + k_lane, stage + t * 1024);
            pg_dma16<ONCE>(vt[t] + v_lane, stage + 32 * ROW + t * 1024);
          }
        } else {
          pg_dma16<ONCE>((l < 32 ? kt[0] : kt[1]) + k_lane, stage + 0);
          pg_dma16<ONCE>((l < 32 ? vt[0] : vt[1]) + v_lane, stage + 32 * ROW);
        }
        if constexpr (NG == 1) {
          const char *k = (l < 16 ? kpt[0] : kpt[1]) + kp_lane, *v = (l < 48 ? vpt[0] : vpt[1]) + vp_lane;
          pg_dma4<ONCE>(l < 32 ? k : v, stage + S::kPairs);
        } else if constexpr (NG == 2) {
          pg_dma4<ONCE>((l < 32 ? kpt[0] : kpt[1]) + kp_lane, stage + S::kPairs);
          pg_dma4<ONCE>((l < 32 ? vpt[0] : vpt[1]) + vp_lane, stage + S::kPairs + 256);
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            pg_dma4<ONCE>(kpt[t] + kp_lane, stage + S::kPairs + t * 256);
            pg_dma4<ONCE>(vpt[t] + vp_lane, stage + S::kPairs + 512 + t * 256);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    uint32_t k_at[NG], v_at[NG]; // of this lane's part of a group in a stage: K, row lq; V, row 4 lg
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int kb = n * (GG / 2) + lg * (GG / 8), vb = n * (GG / 2) + lq * VB;
      k_at[n] = lds + (uint32_t)(lq * ROW + ((kb / 16 ^ swizzle(lq)) << 4) + kb % 16);
      v_at[n] = lds + (uint32_t)(32 * ROW + lg * 4 * ROW + ((vb / 16 ^ swizzle(lg * 4)) << 4) + vb % 16);
    }
    const uint32_t pairs_at = lds + (uint32_t)(S::kPairs + lg * 16 * NG);

    f32x4 o[T];
#pragma unroll
    for (int j = 0; j < T; ++j)
      o[j] = f32x4{0, 0, 0, 0};
    f32x4 z[NG];    // 4 bits: sums of the rounded P scale
    float lows[NG], scales[NG]; // and of P low and of P scale, over this lane's keys
#pragma unroll
    for (int n = 0; n < NG; ++n)
      z[n] = f32x4{0, 0, 0, 0}, lows[n] = scales[n] = 0.f;
    float m = kNegBig, sum = 0.f; // of row lq: maximum of Q . K over all lanes, sum over this lane's keys
    int lift = LIFT ? kLift : 0;  // of row lq, in all of its lanes

    // ---- a chunk's steps: scores, probabilities p, their product with V ---------------------
    float s[8], p[8];
    // in 4 bits the words and pairs of K and V that LDS holds; of group n: tile t's row lq, and key e
    typedef std::conditional_t<SG == 4, u32x4, std::conditional_t<SG == 2, u32x2, uint32_t>> KWords;
    constexpr int kVReads = 8 * NG;
    KWords kw[2][NG];
    uint32_t vw[kVReads];
    u32x4 kpar[2][NG], vpar[2][NG];
    // word r * NG + n of a tile: the pair of this lane's key r, group n
    auto pair_of = [&](u32x4(&x)[2][NG], int t, int r, int n) {
      // (through a scalar: bit-casting a vector's element in place reads element 0)
      const uint32_t w = x[t][(r * NG + n) / 4][(r * NG + n) % 4];
      return __builtin_bit_cast(f16x2, w);
    };
    auto read_pairs = [&](u32x4(&x)[2][NG], uint32_t stage, auto which) {
      pg_static_for<2 * NG>([&](auto ic) {
        constexpr int t = decltype(ic)::value / NG, n = decltype(ic)::value % NG;
        pg_read<decltype(which)::value * 128 * NG + t * 64 * NG + n * 16>(x[t][n], pairs_at + stage);
      });
    };
    auto pin_pairs = [&](u32x4(&x)[2][NG]) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NG; ++n)
          pg_pin(x[t][n]);
    };
    auto read_k = [&](int i) {
      const uint32_t stage = (uint32_t)(i % S::kStages * S::kStage);
      pg_static_for<2 * NG>([&](auto ic) {
        constexpr int t = decltype(ic)::value / NG, n = decltype(ic)::value % NG;
        pg_read<t * 16 * ROW>(kw[t][n], k_at[n] + stage);
      });
      read_pairs(kpar, stage, std::integral_constant<int, 0>{});
    };
    auto read_v = [&](int i) {
      const uint32_t stage = (uint32_t)(i % S::kStages * S::kStage);
      pg_static_for<8 * NG>([&](auto ic) {
        constexpr int n = decltype(ic)::value / 8, e = decltype(ic)::value % 8;
        constexpr int off = ((e >> 2) * 16 + (e & 3)) * ROW;
        if constexpr (VB == 4)
          pg_read<off>(vw[n * 8 + e], v_at[n] + stage);
        else if constexpr (VB == 2)
          pg_read16<off>(vw[n * 8 + e], v_at[n] + stage);
        else
          pg_read8<off>(vw[n * 8 + e], v_at[n] + stage);
      });
      read_pairs(vpar, stage, std::integral_constant<int, 1>{});
    };
    auto wait_k = [&]() {
      pg_lds_wait();
      pin_pairs(kpar);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NG; ++n)
          pg_pin(kw[t][n]);
    };
    auto wait_v = [&]() {
      pg_lds_wait();
      pin_pairs(vpar);
#pragma unroll
      for (int e = 0; e < kVReads; ++e)
        pg_pin(vw[e]);
    };
    auto scores = [&](Chunk &x) {
      if constexpr (Q4) {
        f32x4 a[2][NG]; // (products first: a sum waits for its last one)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            uint32_t w[SG];
            if constexpr (SG == 4)
              w[0] = kw[t][n].x, w[1] = kw[t][n].y, w[2] = kw[t][n].z, w[3] = kw[t][n].w;
            else if constexpr (SG == 2)
              w[0] = kw[t][n].x, w[1] = kw[t][n].y;
            else
              w[0] = kw[t][n];
            // bf16 starts at -128 sum(Q).  f16's 1024 would leave the score 2^-14 of sum |Q| scale:
            // it is taken off the codes
            const float start = BF16 ? -Codes<BF16>::kOffset * qsum[n] : 0.f;
            a[t][n] = f32x4{start, start, start, start};
#pragma unroll
            for (int u = 0; u < SG; ++u) {
              uint32_t f[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                f[e] = codes.pair(w[u], e);
                if constexpr (!BF16)
                  f[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, f[e]) - f16x2{(_Float16)1024, (_Float16)1024});
              }
              a[t][n] = pg_mfma<BF16>(f, qf[n * SG + u], a[t][n]);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              const f16x2 c = pair_of(kpar, t, r, n);
              v = __builtin_fmaf((float)c.x, a[t][n][r], __builtin_fmaf((float)c.y, qsum[n], v));
            }
            s[t * 4 + r] = v;
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 a{0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < KD; ++u) {
            const u32x4 y = x.k[t * KD + u];
            const uint32_t f[4] = {y.x, y.y, y.z, y.w};
            a = pg_mfma<BF16>(f, qf[u], a);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[t * 4 + r] = a[r];
        }
      }
    };
    // The reference point m of the exponentials follows the maximum lazily: a chunk first runs against the one it
    // inherits, with no maximum taken and nothing exchanged between lanes.  Only the first chunk, and one in which
    // some lane's probabilities rise above kRedo, take the maximum and rescale; O = sum(P V) / sum(P) does
    // not depend on m.
    auto rescale = [&](float by) {
      sum *= by;
#pragma unroll
      for (int j = 0; j < T; ++j)
        o[j] *= by;
      if constexpr (Q4)
#pragma unroll
        for (int n = 0; n < NG; ++n)
          z[n] *= by, lows[n] *= by, scales[n] *= by;
    };
    auto softmax = [&](int i, int bad) {
      const int key0 = (c0 + wave + kWaves * i) * kChunk;
      if (bad) { // (the asm keeps this a branch)
        asm volatile("" : "+v"(s[0]));
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s[e] = bad >> (e >> 2) & 1 ? __builtin_nanf("") : s[e];
      }
      if (key0 + kChunk > all_see) {
        int key = key0 + lg * 4;
        asm volatile("" : "+v"(key)); // (and its sums in here)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s[e] = key + (e >> 2) * 16 + (e & 3) < seen ? s[e] : -INFINITY;
      }
      float psum;
      auto exps = [&]() {
        const float at_m = LIFT ? __builtin_fmaf(-m, g.scale_log2e, (float)lift) : -(m * g.scale_log2e);
        psum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], g.scale_log2e, at_m));
          psum += p[e];
        }
      };
      if (i > 0)
        exps();
      if (i == 0 || __builtin_amdgcn_ballot_w64(!(psum <= (LIFT ? __builtin_ldexpf(kRedo, lift) : kRedo))) != 0) {
        float top = s[0];
        asm volatile("" : "+v"(top)); // (keeps the maximum in this branch)
#pragma unroll
        for (int e = 1; e < 8; ++e)
          top = fmaxf(top, s[e]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mn = fmaxf(m, top);
        const int raised = LIFT && mn > m ? kLift - lift : 0;
        const float alpha = __builtin_amdgcn_exp2f(__builtin_fmaf(m - mn, g.scale_log2e, (float)raised));
        m = mn, lift += raised;
        rescale(alpha);
        exps();
      }
      sum += psum;
    };
    // keys behind the last: nothing of theirs may reach a sum
    auto clear_behind = [&](Chunk &x, int i) {
      const int key0 = (c0 + wave + kWaves * i) * kChunk;
      if (key0 + kChunk > keys) {
        int key = key0 + lg * 4;
        asm volatile("" : "+v"(key));
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (key + (e >> 2) * 16 + (e & 3) >= keys) {
            if constexpr (Q4)
#pragma unroll
              for (int n = 0; n < NG; ++n)
                vpar[e >> 2][((e & 3) * NG + n) / 4][((e & 3) * NG + n) % 4] = 0;
            else
              x.v[e] = u32x4{};
          }
      }
    };
    auto values = [&](Chunk &x) {
      if constexpr (Q4) {
        constexpr uint32_t kOne = BF16 ? 0x3f803f80u : 0x3c003c00u;
        const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float ps[8], part = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const f16x2 pr = pair_of(vpar, e >> 2, e & 3, n);
            ps[e] = __builtin_fmaf(p[e], (float)pr.x, 0.f);
            lows[n] = __builtin_fmaf(p[e], (float)pr.y, lows[n]);
            if constexpr (LIFT)
              part += ps[e];
            else
              scales[n] += ps[e];
          }
          if constexpr (LIFT) {
            if (__builtin_amdgcn_ballot_w64(!(part <= kMost)) != 0) {
              float most = part;
              asm volatile("" : "+v"(most)); // (keeps this a branch)
              most = fmaxf(most, __shfl_xor(most, 16, 64));
              most = fmaxf(most, __shfl_xor(most, 32, 64));
              // to between 2^14 and kMost; groups in front of this one have this chunk in their sums already
              const int down = most > kMost && most < INFINITY ? (int)(__builtin_bit_cast(uint32_t, most) >> 23) - (127 + 14) : 0;
              const float by = __builtin_ldexpf(1.0f, -down);
              lift -= down;
              part *= by;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                p[e] *= by, ps[e] *= by;
              rescale(by);
            }
            scales[n] += part;
          }
          const uint32_t pf[4] = {pg_pack<BF16>(ps[0], ps[1]), pg_pack<BF16>(ps[2], ps[3]),
                                  pg_pack<BF16>(ps[4], ps[5]), pg_pack<BF16>(ps[6], ps[7])};
          z[n] = pg_mfma<BF16>(ones, pf, z[n]);
          uint32_t lo[4], hi[4]; // nibbles of the keys 2 e and 2 e + 1 in the halves
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w0 = vw[n * 8 + 2 * e], w1 = vw[n * 8 + 2 * e + 1];
            lo[e] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
            hi[e] = VB == 4 ? __builtin_amdgcn_perm(w1, w0, 0x07060302u) : 0;
          }
#pragma unroll
          for (int j = 0; j < TG; ++j) {
            uint32_t f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[e] = codes.pair(j < 4 ? lo[e] : hi[e], j & 3);
            o[n * TG + j] = pg_mfma<BF16>(f, pf, o[n * TG + j]);
          }
        }
      } else {
        const uint32_t pf[4] = {pg_pack<BF16>(p[0], p[1]), pg_pack<BF16>(p[2], p[3]),
                                pg_pack<BF16>(p[4], p[5]), pg_pack<BF16>(p[6], p[7])};
#pragma unroll
        for (int j = 0; j < T; ++j) {
          uint32_t f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            f[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][j / 2], x.v[2 * e][j / 2],
                                         j & 1 ? 0x07060302u : 0x05040100u);
          o[j] = pg_mfma<BF16>(f, pf, o[j]);
        }
      }
    };
    Chunk x0, x1;
    if constexpr (Q4) {
      for (int i = 0; i < S::kStages - 1 && i < steps; ++i)
        issue(i);
    } else if (steps > 0) {
      fetch(x0, 0);
    }
    if constexpr (Q4) { // (behind the first loads)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float s = 0.f;
#pragma unroll
        for (int u = n * SG; u < (n + 1) * SG; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s += pg_value<BF16>(qf[u][i], 0) + pg_value<BF16>(qf[u][i], 1);
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        qsum[n] = s;
      }
    }
    if constexpr (Q4) {
      // A chunk's words come out of LDS while the step in front of the one that takes them runs: K's beside the last
      // chunk's product with V, V's beside its own scores.  (Four groups' words are too many registers for that.)
      constexpr bool kAhead = NG < 4;
#pragma clang loop unroll(disable)
      for (int i = 0; i < steps; ++i) {
        // (stage (i - 1) % kStages, whose reads the last chunk has waited for)
        if (i + S::kStages - 1 < steps)
          issue(i + S::kStages - 1);
        // chunk i is in LDS when no more than the younger chunks' loads are out
        const int younger = steps - 1 - i < S::kStages - 1 ? steps - 1 - i : S::kStages - 1;
        if (younger == 3)
          __builtin_amdgcn_s_waitcnt(pg_wait_imm(3 * kDmas));
        else if (younger == 2)
          __builtin_amdgcn_s_waitcnt(pg_wait_imm(2 * kDmas));
        else if (younger == 1)
          __builtin_amdgcn_s_waitcnt(pg_wait_imm(kDmas));
        else
          __builtin_amdgcn_s_waitcnt(pg_wait_imm(0));
        asm volatile("" ::: "memory");
        const int bad = (int)(bads >> (2 * younger)) & 3;
        read_k(i);
        __builtin_amdgcn_sched_barrier(0);
        if (kAhead && i > 0)
          values(x0);
        __builtin_amdgcn_sched_barrier(0);
        wait_k();
        if (kAhead)
          read_v(i);
        __builtin_amdgcn_sched_barrier(0);
        scores(x0);
        if (!kAhead)
          read_v(i);
        softmax(i, bad);
        wait_v();
        clear_behind(x0, i);
        if (!kAhead)
          values(x0);
      }
      if (kAhead && steps > 0)
        values(x0);
    } else {
      auto spend = [&](Chunk &x, int i) {
        scores(x);
        softmax(i, x.bad);
        clear_behind(x, i);
        values(x);
      };
      for (int i = 0; i < steps;) {
        if (i + 1 < steps)
          fetch(x1, i + 1);
        spend(x0, i);
        if (++i >= steps)
          break;
        if (i + 1 < steps)
          fetch(x0, i + 1);
        spend(x1, i);
        ++i;
      }
    }

    // ---- the wavefronts' parts meet: O^T value r of tile n * TG + j is column
    // n * GG + (lg * 4 + r) * TG + j of row lq
    const float drop = LIFT ? __builtin_ldexpf(1.0f, -lift) : 1.0f;
    if constexpr (LIFT)
      sum *= drop;
    // (a row that sees no key has a sum below 0, and is 0 whatever values met its probabilities of 0; 0 / 0 stays where all
    // scores that a row sees are -inf)
    sum = beyond ? __builtin_nanf("") : seen == 0 ? -1.f : sum;
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    // The codes' part times the sum of P scale over that of its rounded values: their mean rounding is gone, and with it all
    // of it where one key has (nearly) all of P.
    float even[NG];
    if constexpr (Q4)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        lows[n] = __builtin_fmaf(8.f, scales[n], lows[n]);
        lows[n] += __shfl_xor(lows[n], 16, 64);
        lows[n] += __shfl_xor(lows[n], 32, 64);
        scales[n] += __shfl_xor(scales[n], 16, 64);
        scales[n] += __shfl_xor(scales[n], 32, 64);
        even[n] = z[n][0] > 0.f ? scales[n] / z[n][0] : 1.f;
        if constexpr (LIFT)
          even[n] *= drop, lows[n] *= drop;
      }
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int j = 0; j < TG; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v = o[n * TG + j][r];
          if constexpr (Q4)
            v = __builtin_fmaf(__builtin_fmaf(-(Codes<BF16>::kOffset + 8.f), z[n][r], v), even[n], lows[n]);
          sums[(n * GG + (lg * 4 + r) * TG + j) * PITCH + lq] = v;
        }
    if (l < 16)
      ml[wave][0][l] = m, ml[wave][1][l] = sum;
    __syncthreads();
    const int d = threadIdx.x % HD;
    for (int q = threadIdx.x / HD; q < 16 && q < left; q += kWaves * 64 / HD) {
      float top = ml[0][0][q];
#pragma unroll
      for (int w = 1; w < kWaves; ++w)
        top = fmaxf(top, ml[w][0][q]);
      float acc = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f((ml[w][0][q] - top) * g.scale_log2e);
        acc += ((const float *)(smem + w * S::kBytes))[d * PITCH + q] * f;
        den += ml[w][1][q] * f;
      }
      if (!whole) {
        const int64_t to = ((int64_t)blockIdx.x * 2 + slot) * 16 + q;
        ((PG_AS1 float *)g.part)[to * HD + d] = acc;
        if (d == 0)
          ((PG_AS1 float *)g.part_ml)[to * 2] = top, ((PG_AS1 float *)g.part_ml)[to * 2 + 1] = den;
      } else {
        const int r = qt * 16 + q, p = r / g.group;
        pg_store<BF16>(g.o, (int64_t)(seq.start + p) * g.o_st + (int64_t)(hk * g.group + r - p * g.group) * g.o_sh + d,
                       den < 0.f ? 0.f : acc / den);
      }
    }
    __syncthreads(); // (before the next segment's rows or sums)
  }
}

// Joins the pieces of one row of a query head, which TEAMS of HD threads take in turn: several where there are few rows
// (up to kJoinRows), which may have many pieces each; otherwise one, of 4 columns a thread.  One chat of 30000 keys in 4 bits,
// 117 pieces: 38.8 us with one team, 33.2 with four; 192 rows of 32 heads, few of which have more than three, 110 and 122.
constexpr int kJoinWide = 512, kJoinRows = 512;
template <int HD, int TEAMS> struct JoinShape {
  static constexpr int kVec = TEAMS > 1 ? 1 : 4; // columns of a thread
  static constexpr int kThreads = TEAMS > 1 ? TEAMS * HD : 256;
  static constexpr int kRows = kThreads * kVec / (TEAMS * HD); // rows of a workgroup
};
template <bool BF16, int HD, int TEAMS>
__global__ __launch_bounds__((JoinShape<HD, TEAMS>::kThreads)) void sdpa_paged_join_kernel(PagedArgs g) {
  constexpr int VEC = JoinShape<HD, TEAMS>::kVec, ROWS = JoinShape<HD, TEAMS>::kRows;
  __shared__ float parts[TEAMS][HD], tops[TEAMS], dens[TEAMS];
  const uint32_t heads = (uint32_t)(g.Hkv * g.group);
  const uint32_t lin = blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / (HD / VEC) : 0);
  if (lin >= (uint32_t)g.T * heads)
    return;
  const int d = threadIdx.x % (HD / VEC) * VEC, team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / HD) : 0;
  const int t = (int)(lin / heads), h = (int)(lin % heads);
  const int begins = g.offsets[0], ends = g.offsets[g.cache.batch];
  const PagedArgs::Info info = g.info[t];
  if (t < begins || t >= ends)
    return;
  const int hk = h / g.group;
  if (info.large < 1 || info.small < 1 || info.chunks < 1 || info.pos < 0) // (rows that offsets which overlap have left out hold anything)
    return;
  const uint32_t row = (uint32_t)info.pos * (uint32_t)g.group + (uint32_t)(h - hk * g.group);
  const uint32_t item = (uint32_t)hk * (uint32_t)info.tiles + row / 16;
  const FhipParts parts_of = FhipPieces{info.large, info.small}.parts((uint32_t)info.first + item * (uint32_t)info.chunks,
                                                                      (uint32_t)info.chunks, g.pieces);
  const int begin = parts_of.begin, pieces = parts_of.count;
  if (pieces == 0) // (its one workgroup has stored it)
    return;
  typedef float Vec __attribute__((ext_vector_type(VEC)));
  const PG_AS1 float *ml = (const PG_AS1 float *)g.part_ml;
  const PG_AS1 float *p = (const PG_AS1 float *)g.part;
  struct Part {
    float m, l;
    Vec o;
  };
  const auto load = [&](int s) {
    const int64_t at = ((int64_t)(begin + s) * 2 + (s == 0)) * 16 + row % 16;
    return Part{ml[at * 2], ml[at * 2 + 1], *(const PG_AS1 Vec *)(p + at * HD + d)};
  };
  float top = kNegBig, den = 0.f;
  Vec acc = 0.f;
  const auto take = [&](const Part &x) {
    const float m = fmaxf(top, x.m);
    const float was = __builtin_amdgcn_exp2f((top - m) * g.scale_log2e),
                f = __builtin_amdgcn_exp2f((x.m - m) * g.scale_log2e);
    den = den * was + x.l * f;
    acc = acc * was + x.o * f;
    top = m;
  };
  fhip_for_uniform_parts<(TEAMS > 1 ? 4 : 8)>(team, TEAMS, pieces, load, take);
  if constexpr (TEAMS > 1) { // (all of a workgroup's threads have the same row, and come here or none)
    parts[team][d] = acc[0];
    if (d == 0)
      tops[team] = top, dens[team] = den;
    __syncthreads();
    if (team != 0)
      return;
#pragma unroll
    for (int i = 1; i < TEAMS; ++i)
      take(Part{tops[i], dens[i], Vec{parts[i][d]}});
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    pg_store<BF16>(g.o, (int64_t)t * g.o_st + (int64_t)h * g.o_sh + d + i, den < 0.f ? 0.f : acc[i] / den);
}

// Bytes of K and V that the page table has room for from which they are read as non-temporal: half of what the memory-side
// cache holds.  64 chats of 8192 keys 364 us without, 322 with (4 bits 131.7, 126.1); one of 30000, which the cache keeps from
// call to call, 31.3 and 33.0.  Sequences whose pages are the same, which only the device knows, lose by it: 64 of 4288 keys, 4096 of
// them shared, 84 and 104 us (4 bits 68 and 72); with nothing shared 194 and 172, 32 of 8192 with 1024 shared 169 and 155.
constexpr double kOnce = 128 << 20;
struct PagedPlan {
  bool ok = false;
  int hd = 0, group = 0;
  bool bf16 = false, cut = false, once = false, many = false;
  int64_t pieces = 0; // workgroups
  size_t bytes = 0, part_at = 0, ml_at = 0, upto_at = 0;
};

PagedPlan make_plan(const fhip_sdpa_paged_desc *d) {
  PagedPlan p;
  const int dt = d->q.dtype;
  const int64_t T = d->q.dim[0], Hq = d->q.dim[1], D = d->q.dim[2], Hkv = d->cache.k.dim[1];
  if ((dt != FHIP_BFLOAT16 && dt != FHIP_HALF) || (D != 64 && D != 128) || d->o.dim[2] != D)
    return p;
  if (!fhip_tuned_scale(d->has_scale, d->scale))
    return p;
  p.bf16 = dt == FHIP_BFLOAT16;
  p.hd = (int)D;
  const bool q4 = d->cache.k_params.rank != 0;
  if (q4) {
    p.group = (int)(2 * D / d->cache.k_params.dim[3]);
    if (p.group != 32 && p.group != 64 && p.group != 128)
      return p;
  }
  if (d->cache.k.dim[2] % 16 != 0)
    return p;
  auto fits = [](const fhip_tensor_desc &t, int dims, int64_t step) {
    for (int i = 0; i < dims; ++i)
      if (t.dim[i] > 1 && t.stride[i] % step != 0)
        return false;
    return true;
  };
  const int64_t es = q4 ? 1 : 2;
  if (!fits(d->q, 2, 8) || !fits(d->cache.k, 3, 16 / es) || !fits(d->cache.v, 3, 16 / es) ||
      (q4 && (!fits(d->cache.k_params, 3, 2) || !fits(d->cache.v_params, 3, 2))))
    return p;
  // 32-bit offsets within a tile of 16 keys
  if (d->cache.k.stride[2] * es >= (1 << 26) || d->cache.v.stride[2] * es >= (1 << 26) ||
      (q4 && (d->cache.k_params.stride[2] >= (1 << 25) || d->cache.v_params.stride[2] >= (1 << 25))))
    return p;
  const int64_t group = Hq / Hkv, batch = d->cache.batch;
  // tiles of 16 rows, each sequence's last one short
  const int64_t tiles = Hkv * (T * group / 16 + (batch < T ? batch : T));
  if (T * group >= (1ll << 30) || tiles >= (1ll << 29))
    return p;
  const int64_t keys = d->cache.pages_per_sequence * d->cache.k.dim[2];
  const int64_t row = q4 ? d->cache.k.dim[3] + 2 * d->cache.k_params.dim[3] : 2 * D;
  p.once = T * group <= 16 * batch && 2.0 * (double)(row * Hkv) * (double)batch * (double)keys >= kOnce;
  // (the line's places are 31-bit numbers; the second launch has a thread for each 4 columns of a row)
  p.cut = keys > kWhole && T * Hq <= (1 << 24) && tiles * ((keys + kChunk - 1) / kChunk) < (1ll << 31) - (1 << 24);
  p.pieces = tiles;
  if (p.cut) {
    p.pieces = q4 ? kFhipPieces4 : kFhipPieces16;
    p.part_at = ((size_t)T * sizeof(PagedArgs::Info) + 255) / 256 * 256;
    p.ml_at = p.part_at + (size_t)p.pieces * 2 * 16 * (size_t)D * 4;
    p.bytes = p.ml_at + (size_t)p.pieces * 2 * 16 * 8;
  }
  p.many = batch > kLanes;
  if (p.many) {
    p.upto_at = p.bytes;
    p.bytes += (size_t)batch * 4;
  }
  p.ok = true;
  return p;
}

} // namespace

bool fhip_fast_sdpa_paged_applicable(const fhip_sdpa_paged_desc *d) { return make_plan(d).ok; }

size_t fhip_fast_sdpa_paged_workspace(const fhip_sdpa_paged_desc *d) { return make_plan(d).bytes; }

int fhip_fast_sdpa_paged(fhip_ctx *ctx, const fhip_sdpa_paged_desc *d, const fhip_cache_ptrs *cache, const void *q,
                         const void *offsets, void *o, void *workspace, bool *handled) {
  const PagedPlan p = make_plan(d);
  const uintptr_t rows = (uintptr_t)q | (uintptr_t)cache->k | (uintptr_t)cache->v,
                  pairs = (uintptr_t)cache->k_params | (uintptr_t)cache->v_params;
  *handled = p.ok && (rows & 15) == 0 && (pairs & 3) == 0;
  if (!*handled)
    return 0;
  PagedArgs g{};
  g.q = (const char *)q, g.o = (char *)o, g.offsets = (const int32_t *)offsets;
  g.q_st = d->q.stride[0], g.q_sh = d->q.stride[1], g.o_st = d->o.stride[0], g.o_sh = d->o.stride[1];
  g.cache = fhip_cache_view(d->cache, *cache);
  g.T = (int32_t)d->q.dim[0], g.Hkv = (int32_t)d->cache.k.dim[1], g.group = (int32_t)(d->q.dim[1] / g.Hkv);
  g.causal = d->is_causal != 0;
  g.pieces = (int32_t)p.pieces;
  const float scale = d->has_scale ? d->scale : 1.0f / sqrtf((float)p.hd);
  g.scale_log2e = scale * 1.4426950408889634f;
  if (p.cut) {
    g.info = (PagedArgs::Info *)workspace;
    g.part = (float *)((char *)workspace + p.part_at);
    g.part_ml = (float *)((char *)workspace + p.ml_at);
  }
  if (p.many) {
    g.upto = (int32_t *)((char *)workspace + p.upto_at);
    hipLaunchKernelGGL(sdpa_paged_index_kernel, dim3(1), dim3(1024), 0, ctx->stream, g);
    FHIP_HIP_CHECK(ctx, hipGetLastError());
  }
  fhip_note_kernel(ctx, "sdpa_paged d=%d bits=%d group=%d cut=%d", p.hd, p.group ? 4 : 16, p.group, (int)p.cut);
  auto go = [&](auto bf, auto hd, auto grp) {
    constexpr bool BF = decltype(bf)::value;
    constexpr int HD = decltype(hd)::value, G = decltype(grp)::value;
    constexpr int kLds = kWaves * PagedShape<HD, G>::kBytes;
    auto launch = [&](auto kernel, FhipOncePerDevice &configured) {
      if (kLds > 64 * 1024 && !configured.done(ctx->device)) {
        FHIP_HIP_CHECK(ctx, hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
        configured.mark(ctx->device);
      }
      hipLaunchKernelGGL(kernel, fhip_line_grid(p.pieces), dim3(kWaves * 64), kLds, ctx->stream, g);
      return 0;
    };
    static FhipOncePerDevice configured[2]; // (two for each instance of this lambda)
    if (p.once ? launch(sdpa_paged_kernel<BF, HD, G, true>, configured[0])
               : launch(sdpa_paged_kernel<BF, HD, G, false>, configured[1]))
      return 1;
    if (p.cut) {
      auto join = [&](auto teams) {
        constexpr int TEAMS = decltype(teams)::value, kRows = JoinShape<HD, TEAMS>::kRows;
        const int64_t rows = (int64_t)g.T * g.Hkv * g.group;
        hipLaunchKernelGGL((sdpa_paged_join_kernel<BF, HD, TEAMS>), dim3((unsigned)((rows + kRows - 1) / kRows)),
                           dim3(JoinShape<HD, TEAMS>::kThreads), 0, ctx->stream, g);
      };
      if ((int64_t)g.T * g.Hkv * g.group <= kJoinRows)
        join(std::integral_constant<int, kJoinWide / HD>{});
      else
        join(std::integral_constant<int, 1>{});
    }
    FHIP_HIP_CHECK(ctx, hipGetLastError());
    return 0;
  };
  using std::integral_constant;
  auto grouped = [&](auto bf, auto hd) {
    constexpr int HD = decltype(hd)::value;
    if (p.group == 32)
      return go(bf, hd, integral_constant<int, 32>{});
    if (p.group == 64)
      return go(bf, hd, integral_constant<int, 64>{});
    if constexpr (HD == 128)
      if (p.group == 128)
        return go(bf, hd, integral_constant<int, 128>{});
    return go(bf, hd, integral_constant<int, 0>{});
  };
  auto typed = [&](auto hd) { return p.bf16 ? grouped(std::true_type{}, hd) : grouped(std::false_type{}, hd); };
  return p.hd == 128 ? typed(integral_constant<int, 128>{}) : typed(integral_constant<int, 64>{});
}
