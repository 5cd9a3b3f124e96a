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
// probabilities in f32.  P scale is rounded where P would be: one rounding as in
// 16 bits.  Each product's 32 dims (K) or 16 columns (V) lie within a group.
//
// Work: no one but the device knows the lengths.  Every workgroup reads all of
// them, cuts the sum of all sequences' chunks into about `target` equal pieces
// (whole sequences where they are short), and finds its own piece.  Pieces of one
// sequence meet in the workspace, in a fixed order, in a second kernel.
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
  int32_t causal, target, least; // pieces wanted, chunks that a piece has at least
  float scale_log2e;
  // of sequences in several pieces (null: there are none)
  int32_t *info;  // [T] (first part of the row's sequence, its pieces per tile and head, position)
  float *part;    // [parts][16][HD] sums
  float *part_ml; // [parts][16] (m, l)
  int32_t parts;
};

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

// Nibbles i and i + 4 of a word as two 16-bit numbers, both `kOffset` too large.
template <bool BF16> struct Codes {
  static constexpr float kOffset = BF16 ? 128.f : 1024.f;
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int i) {
    return ((w >> (4 * i)) & 0x000f000fu) | (BF16 ? 0x43004300u : 0x64006400u);
  }
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
  const int a = g.offsets[b], e = g.offsets[b + 1];
  s.start = a < 0 ? 0 : a > g.T ? g.T : a;
  s.rows = (e > g.T ? g.T : e) - s.start;
  s.rows = s.rows < 0 ? 0 : s.rows;
  const int len = g.cache.lengths[b];
  s.length = len < 0 ? 0 : len;
  const int room = g.cache.table_pages * g.cache.page_size; // <= 2^30
  const int keys = s.length < room ? s.length : room;
  s.tiles = (int)(((int64_t)s.rows * g.group + 15) / 16);
  s.chunks = keys ? (keys + kChunk - 1) / kChunk : 1;
  return s;
}

template <bool BF16, int HD, int G>
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
  __shared__ float sums[kWaves][HD * PITCH];
  __shared__ float ml[kWaves][2][16];
  // (scale, low) of 32 keys, K's and V's
  __shared__ __attribute__((aligned(16))) uint32_t params[Q4 ? kWaves : 1][2][Q4 ? 32 * NG : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = threadIdx.x & 63, lq = l & 15, lg = l >> 4;
  const FhipCacheView &c = g.cache;

  // ---- this workgroup's piece ------------------------------------------------
  // (the first 64 sequences stay in the lanes for the second walk)
  const Sequence front = l < c.batch ? pg_sequence(g, l) : Sequence{};
  float work = (float)front.tiles * (float)front.chunks;
  for (int b = l + 64; b < c.batch; b += 64) {
    const Sequence s = pg_sequence(g, b);
    work += (float)s.tiles * (float)s.chunks;
  }
  work = pg_lane(pg_scan(work), 63) * (float)g.Hkv;
  int per = (int)(work / (float)g.target) + 1; // chunks of a piece
  per = per < g.least ? g.least : per;
  int b = -1, index = 0, splits = 1, part = 0; // part: of the sequence's first piece
  Sequence seq{};
  int done = 0, parted = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 64) {
    const Sequence s = b0 == 0 ? front : b0 + l < c.batch ? pg_sequence(g, b0 + l) : Sequence{};
    const int cut = (s.chunks + per - 1) / per, mine = s.tiles * g.Hkv * cut;
    const int upto = pg_scan(mine), parts_upto = pg_scan(cut > 1 ? mine : 0);
    const uint64_t past = __builtin_amdgcn_ballot_w64(done + upto > (int)blockIdx.x);
    if (past) {
      const int at = __builtin_ctzll(past);
      b = b0 + at;
      splits = pg_lane(cut, at);
      index = (int)blockIdx.x - (done + pg_lane(upto - mine, at));
      part = parted + pg_lane(parts_upto, at) - pg_lane(mine, at);
      seq = Sequence{pg_lane(s.start, at), pg_lane(s.rows, at), pg_lane(s.length, at), pg_lane(s.tiles, at),
                     pg_lane(s.chunks, at)};
      break;
    }
    done += pg_lane(upto, 63);
    parted += pg_lane(parts_upto, 63);
  }
  // (the tiles of a head are Hkv * splits workgroups apart, on one XCD where that is a
  // multiple of 8: they read the same keys)
  const int qt = b < 0 ? 0 : index / (g.Hkv * splits), rest = b < 0 ? 0 : index % (g.Hkv * splits);
  const int split = rest / g.Hkv, hk = rest % g.Hkv;
  // (what offsets that overlap could lead to)
  if (b < 0 || index < 0 || qt >= seq.tiles || (splits > 1 && (part < 0 || part + index >= g.parts)))
    return;
  const int room = c.table_pages * c.page_size;
  const int keys = seq.length < room ? seq.length : room;
  const int left = seq.rows * g.group - qt * 16; // of the sequence's packed rows from this tile's first
  const int row = qt * 16 + (lq < left ? lq : left - 1);
  const int pos = row / g.group, hg = row - pos * g.group;
  // keys that this lane's row sees
  int seen = g.causal ? seq.length - seq.rows + pos + 1 : seq.length;
  const bool beyond = seen > keys; // of the page table
  seen = seen < 0 ? 0 : beyond ? keys : seen;
  if (g.info && hk == 0 && split == 0 && threadIdx.x < 16) {
    PG_AS1 int32_t *to = (PG_AS1 int32_t *)g.info + (int64_t)(seq.start + pos) * 3;
    to[0] = part, to[1] = splits, to[2] = pos;
  }

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
    if constexpr (Q4) {
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
  }

  // this workgroup's chunks, up to the last key that any of its rows sees
  int chunks = seq.chunks;
  if (g.causal) {
    const int last = (qt * 16 + (left < 16 ? left : 16) - 1) / g.group;
    int top = seq.length - seq.rows + last + 1;
    top = top > keys ? keys : top < 1 ? 1 : top;
    const int need = (top + kChunk - 1) / kChunk;
    chunks = need < chunks ? need : chunks;
  }
  if (keys == 0)
    chunks = 0;
  const int c0 = (int)((int64_t)chunks * split / splits);
  const int c1 = (int)((int64_t)chunks * (split + 1) / splits);
  const int steps = (c1 - c0 - wave + kWaves - 1) / kWaves; // this wavefront's chunks c0 + wave + 4 i

  // ---- loads -------------------------------------------------------------------
  constexpr int ES = Q4 ? 1 : 2; // bytes per stride unit
  const uint32_t k_slot = (uint32_t)(c.k.slot * ES), v_slot = (uint32_t)(c.v.slot * ES);
  const char *k_head = c.k.data + (int64_t)hk * c.k.head * ES;
  const char *v_head = c.v.data + (int64_t)hk * c.v.head * ES;
  const _Float16 *kp_head = c.k.params + (int64_t)hk * c.k.params_head;
  const _Float16 *vp_head = c.v.params + (int64_t)hk * c.v.params_head;
  int pages = 0, slots = 0; // of tile l & 1 of this wavefront's chunk (i & ~31) + (l >> 1)
  auto look_up = [&](int i) {
    const int key = ((c0 + wave + kWaves * (i + (l >> 1))) * 2 + (l & 1)) * 16;
    const uint32_t n = (uint32_t)key / (uint32_t)c.page_size;
    pages = slots = 0;
    if (key < keys) { // (and so n < table_pages)
      slots = key - (int)n * c.page_size;
      pages = c.table[b * c.table_stride + n];
      pages = (uint32_t)pages < (uint32_t)c.pool_pages ? pages : -1;
    }
  };
  // K: Q4 words of a lane's codes, group after group; V: pairs of keys (2 e, 2 e + 1)
  struct Chunk {
    u32x4 k[2][Q4 ? (KD + 3) / 4 : KD];
    uint32_t v[Q4 ? 8 * NG : 1];
    u32x4 v16[Q4 ? 1 : 8];
    uint32_t kp[2], vp[2];
    int bad;
  };
  constexpr int VB = Q4 ? GG / 32 : 4; // bytes of a V row and group per lane
  static_assert(!Q4 || VB == 4 || VB == 2 || VB == 1, "groups of 32, 64 or 128");
  auto fetch = [&](Chunk &x, int i) {
    if ((i & 31) == 0)
      look_up(i);
    x.bad = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int page = __builtin_amdgcn_readlane(pages, (i & 31) * 2 + t);
      const int slot = __builtin_amdgcn_readlane(slots, (i & 31) * 2 + t);
      if (page < 0)
        page = 0, x.bad |= 1 << t;
      const char *kp = k_head + ((int64_t)page * c.k.page + (int64_t)slot * c.k.slot) * ES;
      const char *vp = v_head + ((int64_t)page * c.v.page + (int64_t)slot * c.v.slot) * ES;
      if constexpr (Q4) {
        uint32_t w[KD];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const char *p = kp + (uint64_t)((uint32_t)lq * k_slot + (uint32_t)(lg * (GG / 8) + n * (GG / 2)));
          if constexpr (SG == 4) {
            const u32x4 y = *(const PG_AS1 u32x4 *)p;
            w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
          } else if constexpr (SG == 2) {
            const u32x2 y = *(const PG_AS1 u32x2 *)p;
            w[n * 2] = y.x, w[n * 2 + 1] = y.y;
          } else {
            w[n] = *(const PG_AS1 uint32_t *)p;
          }
        }
#pragma unroll
        for (int u = 0; u < KD; ++u)
          x.k[t][u / 4][u % 4] = w[u];
        const uint32_t row0 = (uint32_t)(lg * 4) * v_slot + (uint32_t)(lq * VB);
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) { // keys 4 lg + 2 e and + 1 of this tile
            const char *p = vp + (uint64_t)(row0 + (uint32_t)(n * (GG / 2))) + (uint64_t)(2 * e) * v_slot;
            if constexpr (VB == 4) {
              x.v[(t * 2 + e) * 2] = *(const PG_AS1 uint32_t *)p;
              x.v[(t * 2 + e) * 2 + 1] = *(const PG_AS1 uint32_t *)(p + v_slot);
            } else {
              typedef unsigned short us2 __attribute__((ext_vector_type(2)));
              us2 y;
              if constexpr (VB == 2) {
                y.x = *(const PG_AS1 unsigned short *)p;
                y.y = *(const PG_AS1 unsigned short *)(p + v_slot);
              } else {
                y.x = *(const PG_AS1 unsigned char *)p;
                y.y = *(const PG_AS1 unsigned char *)(p + v_slot);
              }
              x.v[n * 4 + t * 2 + e] = __builtin_bit_cast(uint32_t, y);
            }
          }
        // parameters: this tile's 16 keys of K in lanes 0 .. 16 NG - 1 .., one pair per lane
        // (NG 4: two tiles of pairs are 64 lanes each)
        const _Float16 *kpp = kp_head + (int64_t)page * c.k.params_page + (int64_t)slot * c.k.params_slot;
        const _Float16 *vpp = vp_head + (int64_t)page * c.v.params_page + (int64_t)slot * c.v.params_slot;
        if (l < 16 * NG) {
          x.kp[t] = *(const PG_AS1 uint32_t *)(kpp + (int64_t)(l / NG) * c.k.params_slot + l % NG * 2);
          x.vp[t] = *(const PG_AS1 uint32_t *)(vpp + (int64_t)(l / NG) * c.v.params_slot + l % NG * 2);
        }
      } else {
#pragma unroll
        for (int u = 0; u < KD; ++u)
          x.k[t][u] = *(const PG_AS1 u32x4 *)(kp + (uint64_t)((uint32_t)lq * k_slot + (uint32_t)(lg * 16 + u * 64)));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char *p = vp + (uint64_t)((uint32_t)(lg * 4) * v_slot + (uint32_t)(lq * T * 2)) + (uint64_t)r * v_slot;
          if constexpr (T == 8) {
            x.v16[t * 4 + r] = *(const PG_AS1 u32x4 *)p;
          } else {
            const u32x2 y = *(const PG_AS1 u32x2 *)p;
            x.v16[t * 4 + r].x = y.x, x.v16[t * 4 + r].y = y.y;
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  f32x4 o[T];
#pragma unroll
  for (int j = 0; j < T; ++j)
    o[j] = f32x4{0, 0, 0, 0};
  f32x4 z[NG];    // 4 bits: sums of the rounded P scale
  float lows[NG]; // and of P low, over this lane's keys
#pragma unroll
  for (int n = 0; n < NG; ++n)
    z[n] = f32x4{0, 0, 0, 0}, lows[n] = 0.f;
  float m = kNegBig, sum = 0.f; // of row lq: maximum over all lanes, sum over this lane's keys

  auto spend = [&](Chunk &x, int i) {
    const int key0 = (c0 + wave + kWaves * i) * kChunk;
    const bool ends = key0 + kChunk > keys; // keys behind the last: nothing of theirs may reach a sum
    u32x4 kpar[2][NG], vpar[2][NG]; // pairs of this lane's 4 keys of a tile: [t][..] is 4 NG words
    if constexpr (Q4) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (l < 16 * NG) {
          params[wave][0][t * 16 * NG + l] = x.kp[t];
          params[wave][1][t * 16 * NG + l] = x.vp[t];
        }
      // (one wavefront writes and reads: its LDS operations keep their order)
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          kpar[t][n] = *(const u32x4 *)&params[wave][0][(t * 16 + lg * 4) * NG + n * 4];
          vpar[t][n] = *(const u32x4 *)&params[wave][1][(t * 16 + lg * 4) * NG + n * 4];
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    // pair of key r of tile t, group n: word r * NG + n
    auto pair_of = [&](u32x4(&p)[2][NG], int t, int r, int n) {
      // (through a scalar: bit-casting a vector's element in place reads element 0)
      const uint32_t w = p[t][(r * NG + n) / 4][(r * NG + n) % 4];
      return __builtin_bit_cast(f16x2, w);
    };
    float s[8];
    uint32_t live = 0;
    float top = kNegBig;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float v[4];
      if constexpr (Q4) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = 0.f;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          // bf16 starts at -128 sum(Q).  f16's 1024 would leave the score 2^-14 of sum |Q| scale:
          // it is taken off the codes
          const float start = BF16 ? -Codes<BF16>::kOffset * qsum[n] : 0.f;
          f32x4 a{start, start, start, start};
#pragma unroll
          for (int u = n * SG; u < (n + 1) * SG; ++u) {
            const uint32_t w = x.k[t][u / 4][u % 4];
            uint32_t f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] = Codes<BF16>::pair(w, e);
              if constexpr (!BF16)
                f[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, f[e]) - f16x2{(_Float16)1024, (_Float16)1024});
            }
            a = pg_mfma<BF16>(f, qf[u], a);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f16x2 p = pair_of(kpar, t, r, n);
            v[r] = __builtin_fmaf((float)p.x, a[r], __builtin_fmaf((float)p.y, qsum[n], v[r]));
          }
        }
      } else {
        f32x4 a{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < KD; ++u) {
          const u32x4 y = x.k[t][u];
          const uint32_t f[4] = {y.x, y.y, y.z, y.w};
          a = pg_mfma<BF16>(f, qf[u], a);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = a[r];
      }
      if (x.bad & (1 << t))
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = __builtin_nanf("");
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = key0 + t * 16 + lg * 4 + r < seen;
        live |= (uint32_t)in << (t * 4 + r);
        s[t * 4 + r] = v[r] * g.scale_log2e;
        top = fmaxf(top, in ? s[t * 4 + r] : kNegBig);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top);
    if (__builtin_amdgcn_ballot_w64(mn > m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      sum *= alpha;
#pragma unroll
      for (int j = 0; j < T; ++j)
        o[j] *= alpha;
      if constexpr (Q4)
#pragma unroll
        for (int n = 0; n < NG; ++n)
          z[n] *= alpha, lows[n] *= alpha;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = (live >> e) & 1 ? __builtin_amdgcn_exp2f(s[e] - m) : 0.f;
      sum += p[e];
    }
    if constexpr (Q4) {
      if (ends)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + t * 16 + lg * 4 + r >= keys)
#pragma unroll
              for (int n = 0; n < NG; ++n)
                vpar[t][(r * NG + n) / 4][(r * NG + n) % 4] = 0;
      constexpr uint32_t kOne = BF16 ? 0x3f803f80u : 0x3c003c00u;
      const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float ps[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const f16x2 pr = pair_of(vpar, e >> 2, e & 3, n);
          ps[e] = p[e] * (float)pr.x;
          lows[n] = __builtin_fmaf(p[e], (float)pr.y, lows[n]);
        }
        const uint32_t pf[4] = {pg_pack<BF16>(ps[0], ps[1]), pg_pack<BF16>(ps[2], ps[3]),
                                pg_pack<BF16>(ps[4], ps[5]), pg_pack<BF16>(ps[6], ps[7])};
        z[n] = pg_mfma<BF16>(ones, pf, z[n]);
        uint32_t lo[4], hi[4]; // nibbles of the keys 2 e and 2 e + 1 in the halves
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (VB == 4) {
            lo[e] = __builtin_amdgcn_perm(x.v[2 * e + 1], x.v[2 * e], 0x05040100u);
            hi[e] = __builtin_amdgcn_perm(x.v[2 * e + 1], x.v[2 * e], 0x07060302u);
          } else {
            lo[e] = x.v[n * 4 + e];
            hi[e] = 0;
          }
        }
#pragma unroll
        for (int j = 0; j < TG; ++j) {
          uint32_t f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            f[e] = Codes<BF16>::pair(j < 4 ? lo[e] : hi[e], j & 3);
          o[n * TG + j] = pg_mfma<BF16>(f, pf, o[n * TG + j]);
        }
      }
    } else {
      if (ends)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (key0 + (e >> 2) * 16 + lg * 4 + (e & 3) >= keys)
            x.v16[e] = u32x4{};
      const uint32_t pf[4] = {pg_pack<BF16>(p[0], p[1]), pg_pack<BF16>(p[2], p[3]),
                              pg_pack<BF16>(p[4], p[5]), pg_pack<BF16>(p[6], p[7])};
#pragma unroll
      for (int j = 0; j < T; ++j) {
        uint32_t f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f[e] = __builtin_amdgcn_perm(x.v16[2 * e + 1][j / 2], x.v16[2 * e][j / 2],
                                       j & 1 ? 0x07060302u : 0x05040100u);
        o[j] = pg_mfma<BF16>(f, pf, o[j]);
      }
    }
  };
  Chunk x0, x1;
  int i = 0;
  if (steps > 0)
    fetch(x0, 0);
  while (i < steps) {
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

  // ---- the wavefronts' parts meet: O^T value r of tile n * TG + j is column
  // n * GG + (lg * 4 + r) * TG + j of row lq
  if (beyond)
    sum = __builtin_nanf("");
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if constexpr (Q4)
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      lows[n] += __shfl_xor(lows[n], 16, 64);
      lows[n] += __shfl_xor(lows[n], 32, 64);
    }
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int j = 0; j < TG; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = o[n * TG + j][r];
        if constexpr (Q4)
          v = __builtin_fmaf(-Codes<BF16>::kOffset, z[n][r], v) + lows[n];
        sums[wave][(n * GG + (lg * 4 + r) * TG + j) * PITCH + lq] = v;
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
      const float f = __builtin_amdgcn_exp2f(ml[w][0][q] - top);
      acc += sums[w][d * PITCH + q] * f;
      den += ml[w][1][q] * f;
    }
    if (splits > 1) {
      const int64_t at = (int64_t)(part + index) * 16 + q;
      ((PG_AS1 float *)g.part)[at * HD + d] = acc;
      if (d == 0)
        ((PG_AS1 float *)g.part_ml)[at * 2] = top, ((PG_AS1 float *)g.part_ml)[at * 2 + 1] = den;
    } else {
      const int r = qt * 16 + q, p = r / g.group;
      pg_store<BF16>(g.o, (int64_t)(seq.start + p) * g.o_st + (int64_t)(hk * g.group + r - p * g.group) * g.o_sh + d,
                     den == 0.f ? 0.f : acc / den);
    }
  }
}

// Joins the pieces of one row of a query head per HD threads.
template <bool BF16, int HD>
__global__ __launch_bounds__(256) void sdpa_paged_join_kernel(PagedArgs g) {
  const uint32_t heads = (uint32_t)(g.Hkv * g.group);
  const uint32_t lin = blockIdx.x * (256 / HD) + threadIdx.x / HD;
  const int d = threadIdx.x % HD;
  if (lin >= (uint32_t)g.T * heads)
    return;
  const int t = (int)(lin / heads), h = (int)(lin % heads);
  if (t < g.offsets[0] || t >= g.offsets[g.cache.batch])
    return;
  const PG_AS1 int32_t *info = (const PG_AS1 int32_t *)g.info + (int64_t)t * 3;
  const int first = info[0], splits = info[1], pos = info[2];
  const int hk = h / g.group;
  const int64_t row = (int64_t)pos * g.group + h - hk * g.group;
  const int64_t piece = first + row / 16 * g.Hkv * splits + hk;
  // (rows that offsets which overlap have left out hold anything)
  if (splits <= 1 || pos < 0 || first < 0 || piece + (int64_t)(splits - 1) * g.Hkv >= g.parts)
    return;
  const PG_AS1 float *ml = (const PG_AS1 float *)g.part_ml;
  const PG_AS1 float *p = (const PG_AS1 float *)g.part;
  struct Part {
    float m, l, o;
  };
  const auto load = [&](int s) {
    const int64_t at = (piece + (int64_t)s * g.Hkv) * 16 + row % 16;
    return Part{ml[at * 2], ml[at * 2 + 1], p[at * HD + d]};
  };
  constexpr int U = 8;
  float top = kNegBig, acc = 0.f, den = 0.f;
  fhip_for_uniform_parts<U>(0, 1, splits, load, [&](const Part &x) {
    const float m = fmaxf(top, x.m);
    const float was = __builtin_amdgcn_exp2f(top - m), f = __builtin_amdgcn_exp2f(x.m - m);
    den = den * was + x.l * f;
    acc = acc * was + x.o * f;
    top = m;
  });
  pg_store<BF16>(g.o, (int64_t)t * g.o_st + (int64_t)h * g.o_sh + d, den == 0.f ? 0.f : acc / den);
}

// Pieces that the work is cut into.
constexpr int kTarget = 512;
// Chunks that a piece has at least, and keys up to which no sequence is cut (the
// launch that joins pieces takes longer than what it saves).
constexpr int kLeast = 2 * kWaves;
constexpr int64_t kWhole = 1024;

struct PagedPlan {
  bool ok = false;
  int hd = 0, group = 0;
  bool bf16 = false, cut = false;
  int64_t pieces = 0, parts = 0;
  size_t bytes = 0, part_at = 0, ml_at = 0;
};

PagedPlan make_plan(const fhip_sdpa_paged_desc *d) {
  PagedPlan p;
  const int dt = d->q.dtype;
  const int64_t T = d->q.dim[0], Hq = d->q.dim[1], D = d->q.dim[2], Hkv = d->cache.k.dim[1];
  if ((dt != FHIP_BFLOAT16 && dt != FHIP_HALF) || (D != 64 && D != 128) || d->o.dim[2] != D)
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
  if (d->cache.k.stride[2] * es >= (1 << 26) || d->cache.v.stride[2] * es >= (1 << 26))
    return p;
  const int64_t group = Hq / Hkv, batch = d->cache.batch;
  // tiles of 16 rows, each sequence's last one short
  const int64_t tiles = Hkv * (T * group / 16 + (batch < T ? batch : T));
  if (T * group >= (1ll << 30) || tiles >= (1ll << 29))
    return p;
  p.cut = d->cache.pages_per_sequence * d->cache.k.dim[2] > kWhole;
  p.pieces = tiles + (p.cut ? kTarget + 8 : 0);
  if (p.cut) {
    // a sequence in several pieces has more chunks than a piece: at most twice kTarget of them
    p.parts = 2 * kTarget + 64;
    p.part_at = ((size_t)T * 12 + 255) / 256 * 256;
    p.ml_at = p.part_at + (size_t)p.parts * 16 * (size_t)D * 4;
    p.bytes = p.ml_at + (size_t)p.parts * 16 * 8;
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
  g.target = kTarget, g.least = p.cut ? kLeast : 1 << 26;
  const float scale = d->has_scale ? d->scale : 1.0f / sqrtf((float)p.hd);
  g.scale_log2e = scale * 1.4426950408889634f;
  if (p.cut) {
    g.info = (int32_t *)workspace;
    g.part = (float *)((char *)workspace + p.part_at);
    g.part_ml = (float *)((char *)workspace + p.ml_at);
    g.parts = (int32_t)p.parts;
  }
  fhip_note_kernel(ctx, "sdpa_paged d=%d bits=%d group=%d cut=%d", p.hd, p.group ? 4 : 16, p.group, (int)p.cut);
  auto go = [&](auto bf, auto hd, auto grp) {
    constexpr bool BF = decltype(bf)::value;
    constexpr int HD = decltype(hd)::value, G = decltype(grp)::value;
    hipLaunchKernelGGL((sdpa_paged_kernel<BF, HD, G>), dim3((unsigned)p.pieces), dim3(kWaves * 64), 0, ctx->stream, g);
    if (p.cut)
      hipLaunchKernelGGL((sdpa_paged_join_kernel<BF, HD>),
                         dim3((unsigned)(((int64_t)g.T * g.Hkv * g.group + 256 / HD - 1) / (256 / HD))), dim3(256), 0,
                         ctx->stream, g);
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
