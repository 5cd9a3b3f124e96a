// Which rows of packed tensors a sequence has, as kernels find it from device memory that no call has
// checked, and where the line of a paged call's chunks is cut: plain arithmetic, the same on the host
// (tests/cpp/test_serving_split.cpp).
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

// ---- the line of chunks --------------------------------------------------------------
// Workgroups that share the line: two for each compute unit run at once.  In 4 bits, where a compute unit has more to
// compute, their ends lie further apart, and 256 more with pieces of a quarter go where one is done: 6 batches of 64 chats
// with drafts 112.3 us in the mean with 512 equal pieces, 112.1 with 1024, 107.0 with 512 and 512 quarters, 107.6 like this.
constexpr int kFhipLargePieces = 512, kFhipPieces16 = kFhipLargePieces, kFhipPieces4 = kFhipLargePieces + 256;
constexpr int kFhipQuarter = 4;
// One round where pieces are fewer chunks than this: 8 chats of 8192 keys 31.2 us in two equal rounds, 25.5 in one.
constexpr int kFhipSmallPiece = 64;
constexpr int kFhipLeastPiece = 8; // chunks that a piece has at least: two for each wavefront
// A cut moves by up to a piece / kFhipNear: 5 batches of 32 chats in 16 bits took 73 .. 90 us with 4, 66 .. 87 with 8,
// 66 .. 85 with 16, of 64 in 4 bits with drafts 102 .. 126, 99 .. 122 and 100 .. 123.
constexpr int kFhipNear = 8;
static_assert(kFhipLeastPiece >= kFhipNear, "a cut at a segment's end is always near");

// The pieces that share a segment, `count` of them from `begin` on; 0: one has all of it.
struct FhipParts {
  int32_t begin, count;
};

// The pieces' places on the line: kFhipLargePieces large ones, then small ones.
struct FhipPieces {
  int32_t large, small; // chunks of each
  static FHIP_SPLIT_FN FhipPieces of(int total, int pieces) {
    const int rest = total < pieces * kFhipSmallPiece ? 0 : pieces - kFhipLargePieces;
    FhipPieces p;
    p.large = (int)(((int64_t)total * kFhipQuarter - 1) / (kFhipLargePieces * kFhipQuarter + rest)) + 1;
    p.large = p.large < kFhipLeastPiece ? kFhipLeastPiece : p.large;
    p.small = (p.large + kFhipQuarter - 1) / kFhipQuarter;
    p.small = p.small < kFhipLeastPiece ? kFhipLeastPiece : p.small;
    return p;
  }
  FHIP_SPLIT_FN int64_t at(uint32_t i) const {
    return i <= kFhipLargePieces ? (int64_t)i * large
                                 : (int64_t)kFhipLargePieces * large + (int64_t)(i - kFhipLargePieces) * small;
  }
  // Where the cut at x goes, in a line of segments of `chunks` from `first` on: to an end of its segment that is near.
  FHIP_SPLIT_FN int moved(int x, int first, int chunks) const {
    const int near = large / kFhipNear, inside = (x - first) % chunks;
    return inside < near ? x - inside : chunks - inside < near ? x - inside + chunks : x;
  }
  // The last piece that begins at x or in front of it (places on the line are 31-bit numbers).
  FHIP_SPLIT_FN uint32_t last(uint32_t x) const {
    const uint32_t bend = (uint32_t)kFhipLargePieces * (uint32_t)large;
    return x < bend ? x / (uint32_t)large : kFhipLargePieces + (x - bend) / (uint32_t)small;
  }
  // What of `pieces` share the segment of `chunks` at `from`: those whose cuts lie inside it and not near its ends, and the
  // one in front.  (Of a line that is none, as overlapping offsets may leave it, still a range of pieces, or none.)
  FHIP_SPLIT_FN FhipParts parts(uint32_t from, uint32_t chunks, int pieces) const {
    const uint32_t near = (uint32_t)large / kFhipNear;
    const int64_t begin = last(from + near - 1), count = (int64_t)last(from + chunks - near) - begin + 1;
    if (chunks < 2 * near || count <= 1 || begin + count > pieces)
      return FhipParts{0, 0};
    return FhipParts{(int32_t)begin, (int32_t)count};
  }
};

#endif // FUSILLI_AMD_CSRC_SERVING_SPLIT_H
