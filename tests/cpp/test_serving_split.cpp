// Which rows a sequence has (fusilli_amd/csrc/serving_split.h), on the host.
#include "../../fusilli_amd/csrc/serving_split.h"
#include "mini_test.h"

#include <algorithm>
#include <climits>

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

int main(int argc, char **argv) { return mini::run(argc, argv); }
