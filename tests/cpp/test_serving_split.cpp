// Which rows a sequence has and where the line of chunks is cut (fusilli_amd/csrc/serving_split.h), on the host.
#include "../../fusilli_amd/csrc/serving_split.h"
#include "mini_test.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <random>
#include <vector>

TEST("offsets of any value stay inside the tensor") {
  const int32_t values[] = {INT_MIN, INT_MIN + 1, INT_MIN + 5, -1000000, -1, 0, 1, 5, 6, 7, 1000000, INT_MAX - 1, INT_MAX};
  for (int32_t T : {1, 6, 1 << 20, INT_MAX - 1})
    for (int32_t begin : values)
      for (int32_t end : values) {
        const FhipRows r = fhip_rows_between(begin, end, T);
        CHECK(r.first >= 0 && r.first <= T && r.count >= 0 && r.count <= T - r.first);
        const int64_t a = std::clamp<int64_t>(begin, 0, T), e = std::clamp<int64_t>(end, 0, T);
        CHECK(r.count == std::max<int64_t>(e - a, 0));
        if (r.count)
          CHECK(r.first == a);
      }
}

namespace {
// A sequence's part of the line: `segments` of `chunks` each, from `first` on.
struct Part {
  int first, chunks, segments;
};
struct Line {
  std::vector<Part> parts;
  int total = 0;
  void add(int chunks, int segments) {
    parts.push_back({total, chunks, segments});
    total += chunks * segments;
  }
};
struct Piece {
  int index, from, to; // chunks of the segment
};

// What the pieces do, as the workgroups go through them, against what the join takes for it.
void check(const Line &line, int pieces) {
  const FhipPieces cut = FhipPieces::of(line.total, pieces);
  CHECK(cut.at(pieces) >= line.total);
  size_t at_part = 0;
  auto part_of = [&](int x) -> const Part & {
    while (x >= line.parts[at_part].first + line.parts[at_part].chunks * line.parts[at_part].segments)
      ++at_part;
    while (x < line.parts[at_part].first)
      --at_part;
    return line.parts[at_part];
  };
  auto end_of = [&](int64_t x) {
    if (x >= line.total)
      return line.total;
    const Part &p = part_of(static_cast<int>(x));
    return cut.moved(static_cast<int>(x), p.first, p.chunks);
  };
  std::vector<Piece> own; // the pieces of the segment that the walk is in
  int covered = 0;
  for (int i = 0; i < pieces; ++i) {
    int at = end_of(cut.at(i));
    const int stop = end_of(cut.at(i + 1));
    CHECK(at == covered && stop >= at);
    bool began = false, went_on = false; // the two places that a piece has for its parts
    while (at < stop) {
      const Part &p = part_of(at);
      const int inside = (at - p.first) % p.chunks, to = std::min(p.chunks, inside + stop - at);
      const bool whole = inside == 0 && to == p.chunks;
      if (!whole) {
        bool &place = inside == 0 ? began : went_on;
        CHECK(!place);
        place = true;
      }
      own.push_back({i, inside, to});
      if (to == p.chunks) {
        const FhipParts parts = cut.parts(at - inside, p.chunks, pieces);
        if (own.size() == 1) {
          CHECK(parts.count == 0);
        } else {
          CHECK(parts.begin == own[0].index && parts.count == static_cast<int>(own.size()));
          for (size_t s = 0; s < own.size(); ++s)
            CHECK(own[s].index == parts.begin + static_cast<int>(s) && (own[s].from == 0) == (s == 0));
        }
        own.clear();
      }
      at += to - inside;
    }
    covered = stop;
  }
  CHECK(covered == line.total && own.empty());
}
} // namespace

TEST("pieces cover the line once, and the join finds them") {
  std::mt19937 rng(1);
  auto pick = [&](int64_t lo, int64_t hi) { // over the logarithm
    std::uniform_real_distribution<double> d(std::log(double(lo)), std::log(double(hi) + 1));
    return static_cast<int>(std::clamp<int64_t>(static_cast<int64_t>(std::exp(d(rng))), lo, hi));
  };
  bool near = false, small = false, behind = false; // cuts that move, small pieces, pieces that have none
  for (int pieces : {kFhipPieces16, kFhipPieces4})
    for (int round = 0; round < 600; ++round) {
      Line line;
      const int longest = pick(1, 1 << pick(1, 20)), sequences = pick(1, 300);
      while (static_cast<int>(line.parts.size()) < sequences && line.total < (1 << 30))
        line.add(round % 3 ? pick(1, longest) : longest, pick(1, 64));
      check(line, pieces);
      const FhipPieces cut = FhipPieces::of(line.total, pieces);
      near |= cut.large / kFhipNear > 1, small |= cut.at(kFhipLargePieces) < line.total, behind |= cut.at(pieces - 1) >= line.total;
    }
  CHECK(near && small && behind);
}

TEST("the longest line") {
  for (int pieces : {kFhipPieces16, kFhipPieces4}) {
    Line one, many;
    one.add(INT_MAX - (1 << 24), 1);
    check(one, pieces);
    while (many.total < INT_MAX - (1 << 25))
      many.add((1 << 18) + 13, 31);
    check(many, pieces);
  }
}

TEST("parts of what is no line are pieces that there are, or none") {
  std::mt19937 rng(2);
  auto any = [&] {
    const uint32_t x = rng();
    return x >> rng() % 32;
  };
  for (int i = 0; i < 2000000; ++i) {
    const FhipPieces cut{static_cast<int32_t>(std::max(1u, any() & 0x7fffffffu)), static_cast<int32_t>(std::max(1u, any() & 0x7fffffffu))};
    const int pieces = i % 2 ? kFhipPieces16 : kFhipPieces4;
    const FhipParts p = cut.parts(any(), std::max(1u, any()), pieces);
    if (p.count)
      CHECK(p.begin >= 0 && p.count > 1 && p.begin + p.count <= pieces);
    else
      CHECK(p.begin == 0);
  }
}

int main(int argc, char **argv) { return mini::run(argc, argv); }
