// Packed sequences and paged caches through the graph API.  "host" cases need no
// GPU: what the nodes check, what a plan holds.  The others run a prompt, a chunk
// behind it and a token through one graph each against plain loops in double.
#include <fusilli.h>

#include <cmath>
#include <random>

#include "mini_test.h"

using namespace fusilli;
using Dims = std::vector<int64_t>;
using Pack = std::unordered_map<std::shared_ptr<TensorAttr>, std::shared_ptr<Buffer>>;

static Dims contig(const Dims &d) {
  return generateStrideFromDim(d, getContiguousStrideOrder(d.size()));
}
static TensorAttr mk(const std::string &name, Dims dim, DataType dt) {
  return TensorAttr().setName(name).setDim(dim).setStride(contig(dim)).setDataType(dt);
}
static Graph newGraph(const std::string &name) {
  Graph g;
  g.setName(name).setIODataType(DataType::BFloat16).setIntermediateDataType(DataType::BFloat16)
      .setComputeDataType(DataType::Float);
  return g;
}

constexpr int64_t kPool = 12, kHq = 4, kHk = 2, kPage = 16, kD = 64, kBatch = 2, kTable = 4, kPlaces = 64;

static CacheTensors cacheOf(Graph &g, int64_t group = 0) {
  CacheTensors c;
  const DataType dt = group ? DataType::Uint8 : DataType::BFloat16;
  const int64_t row = group ? kD / 2 : kD;
  c.k = g.tensor(mk("cache_k", {kPool, kHk, kPage, row}, dt));
  c.v = g.tensor(mk("cache_v", {kPool, kHk, kPage, row}, dt));
  if (group) {
    c.kParams = g.tensor(mk("cache_kp", {kPool, kHk, kPage, 2 * kD / group}, DataType::Half));
    c.vParams = g.tensor(mk("cache_vp", {kPool, kHk, kPage, 2 * kD / group}, DataType::Half));
  }
  c.pages = g.tensor(mk("pages", {kBatch, kTable}, DataType::Int32));
  c.lengths = g.tensor(mk("lengths", {kBatch}, DataType::Int32));
  return c;
}
struct Rows {
  TensorPtr q, k, v, offsets, rotation;
};
static Rows rowsOf(Graph &g, int64_t t) {
  return {g.tensor(mk("q", {t, kHq, kD}, DataType::BFloat16)), g.tensor(mk("k", {t, kHk, kD}, DataType::BFloat16)),
          g.tensor(mk("v", {t, kHk, kD}, DataType::BFloat16)), g.tensor(mk("offsets", {kBatch + 1}, DataType::Int32)),
          g.tensor(mk("rotation", {kPlaces, kD}, DataType::Float))};
}

TEST("host: nodes check their tensors") {
  auto packed = [](auto &&change) {
    Graph g = newGraph("packed");
    Rows r = rowsOf(g, 20);
    TensorPtr kvOffsets;
    change(g, r, kvOffsets);
    SdpaPackedAttr a;
    a.setName("p").setIsCausal(true);
    g.sdpaPacked(r.q, r.k, r.v, r.offsets, kvOffsets, a)->setOutput(true);
    return g.validate();
  };
  REQUIRE_OK(packed([](Graph &, Rows &, TensorPtr &) {}));
  CHECK_ERROR(packed([](Graph &, Rows &r, TensorPtr &) { r.k = nullptr; }), ErrorCode::AttributeNotSet,
              "SDPA packed tensor K not set");
  CHECK_ERROR(packed([](Graph &g, Rows &r, TensorPtr &) { r.q = g.tensor(mk("q4", {1, 20, kHq, kD}, DataType::BFloat16)); }),
              ErrorCode::InvalidAttribute, "SDPA packed tensor Q must be rank 3 [rows, heads, head_dim]");
  CHECK_ERROR(packed([](Graph &g, Rows &r, TensorPtr &) { r.q = g.tensor(mk("q3", {20, 3, kD}, DataType::BFloat16)); }),
              ErrorCode::InvalidAttribute, "SDPA packed requires Q heads (3) to be a multiple of K heads (2)");
  CHECK_ERROR(packed([](Graph &g, Rows &r, TensorPtr &) { r.offsets = g.tensor(mk("o64", {3}, DataType::Int64)); }),
              ErrorCode::InvalidAttribute, "SDPA packed tensor OFFSETS must be Int32");
  CHECK_ERROR(packed([](Graph &g, Rows &, TensorPtr &kv) { kv = g.tensor(mk("kv", {4}, DataType::Int32)); }),
              ErrorCode::InvalidAttribute, "SDPA packed tensor KV_OFFSETS must be contiguous [3]");

  auto paged = [](auto &&change) {
    Graph g = newGraph("paged");
    Rows r = rowsOf(g, 2);
    CacheTensors c = cacheOf(g);
    change(g, r, c);
    SdpaPagedAttr a;
    a.setName("p");
    g.sdpaPaged(r.q, r.offsets, c, a)->setOutput(true);
    return g.validate();
  };
  REQUIRE_OK(paged([](Graph &, Rows &, CacheTensors &) {}));
  CHECK_ERROR(paged([](Graph &, Rows &, CacheTensors &c) { c.pages = nullptr; }), ErrorCode::AttributeNotSet,
              "SDPA paged cache tensors CACHE_K, CACHE_V, PAGES and LENGTHS must be set");
  CHECK_ERROR(paged([](Graph &g, Rows &, CacheTensors &c) { c.lengths = g.tensor(mk("l3", {3}, DataType::Int32)); }),
              ErrorCode::InvalidAttribute, "SDPA paged tensor LENGTHS must be contiguous [2]");
  CHECK_ERROR(paged([](Graph &g, Rows &r, CacheTensors &) { r.offsets = g.tensor(mk("o2", {2}, DataType::Int32)); }),
              ErrorCode::InvalidAttribute, "SDPA paged tensor OFFSETS must be contiguous [3]");
  CHECK_ERROR(paged([](Graph &g, Rows &, CacheTensors &c) {
                c.kParams = g.tensor(mk("kp", {kPool, kHk, kPage, 4}, DataType::Half));
              }),
              ErrorCode::AttributeNotSet, "SDPA paged cache parameters go together");

  Graph g = newGraph("read");
  CacheReadAttr ra;
  ra.setName("r");
  auto kv = g.cacheRead(g.tensor(mk("offsets", {kBatch + 1}, DataType::Int32)), cacheOf(g), ra);
  kv[0]->setOutput(true);
  kv[1]->setOutput(true);
  CHECK_ERROR(g.validate(), ErrorCode::InvalidAttribute,
              "Cache read tensor K must be rank 3 [rows, heads, head_dim]");
}

TEST("host: a step of decoding is two kernels, its rows between them in the workspace; an unread K_OUT is not written") {
  Graph g = newGraph("decode");
  Rows r = rowsOf(g, 2);
  CacheTensors c = cacheOf(g, 32);
  CacheAppendAttr aa;
  auto [qo, ko] = g.cacheAppend(r.q, r.k, r.v, r.rotation, nullptr, r.offsets, c, aa);
  SdpaPagedAttr pa;
  auto o = g.sdpaPaged(qo, r.offsets, c, pa);
  o->setOutput(true);
  REQUIRE_OK(g.validate());
  REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
  REQUIRE_OK(g.compile(cpu, true));
  CHECK(g.getKernelCount() == std::optional<size_t>(2));
  auto ws = g.getWorkspaceSize();
  REQUIRE(!isError(ws) && ws->has_value());
  CHECK(**ws == 2 * kHq * kD * 2); // Q_OUT (the table has room for 64 keys: no parts)
  CHECK(o->getDim() == (Dims{2, kHq, kD}));
  CHECK(ko->isVirtual());
}

TEST("host: keys alone go into a cache; their turned rows are an output where they are marked as one") {
  for (bool out : {false, true}) {
    Graph g = newGraph("prefill");
    Rows r = rowsOf(g, 20);
    CacheTensors c = cacheOf(g);
    CacheAppendAttr aa;
    aa.setName("a");
    auto [qo, ko] = g.cacheAppend(nullptr, r.k, r.v, r.rotation, nullptr, r.offsets, c, aa);
    CHECK(!qo);
    ko->setOutput(out);
    REQUIRE_OK(g.validate());
    REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
    REQUIRE_OK(g.compile(cpu, true));
    CHECK(g.getKernelCount() == std::optional<size_t>(1));
    CHECK(ko->getDim() == (Dims{20, kHk, kD}));
    CHECK(ko->isVirtual() == !out);
  }
}

TEST("host: what no kernel takes is refused by compile") {
  Graph g = newGraph("refused");
  Rows r = rowsOf(g, 2);
  CacheTensors c = cacheOf(g);
  c.k = g.tensor(mk("cache_k32", {kPool, kHk, kPage, kD}, DataType::Float));
  SdpaPagedAttr pa;
  pa.setName("p");
  g.sdpaPaged(r.q, r.offsets, c, pa)->setOutput(true);
  REQUIRE_OK(g.validate());
  REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
  CHECK_ERROR(g.compile(cpu, true), ErrorCode::NotImplemented,
              "SDPA paged node 'p' is not executable by this backend: fhip_sdpa_paged_fwd: the cache's K and V differ "
              "in type");
}

TEST("host: K and caches without heads are refused") {
  for (int64_t heads : {0, -1}) {
    Graph g = newGraph("headless");
    Rows r = rowsOf(g, 20);
    SdpaPackedAttr a;
    a.setName("p");
    g.sdpaPacked(r.q, g.tensor(mk("k0", {20, heads, kD}, DataType::BFloat16)), r.v, r.offsets, nullptr, a)->setOutput(true);
    CHECK_ERROR(g.validate(), ErrorCode::InvalidAttribute,
                "SDPA packed requires Q heads (4) to be a multiple of K heads (" + std::to_string(heads) + ")");
    Graph h = newGraph("headless_cache");
    Rows s = rowsOf(h, 2);
    CacheTensors c = cacheOf(h);
    c.k = h.tensor(mk("cache_k0", {kPool, heads, kPage, kD}, DataType::BFloat16));
    SdpaPagedAttr b;
    b.setName("a");
    h.sdpaPaged(s.q, s.offsets, c, b)->setOutput(true);
    CHECK_ERROR(h.validate(), ErrorCode::InvalidAttribute,
                "SDPA paged requires Q heads (4) to be a multiple of K heads (" + std::to_string(heads) + ")");
  }
}

// ---- on the GPU ----------------------------------------------------------------
static Handle &gpu() {
  static Handle h = [] {
    auto e = Handle::create(Backend::AMDGPU);
    if (isError(e)) {
      std::printf("no AMDGPU handle: %s\n", ErrorObject(e).getMessage().c_str());
      std::exit(2);
    }
    return std::move(*e);
  }();
  return h;
}
template <typename T> static std::shared_ptr<Buffer> bufOf(const std::vector<T> &data, const Dims &dims) {
  auto b = Buffer::allocate(gpu(), std::vector<size_t>(dims.begin(), dims.end()), data);
  if (isError(b)) {
    std::printf("allocate failed: %s\n", ErrorObject(b).getMessage().c_str());
    std::exit(3);
  }
  return std::make_shared<Buffer>(std::move(*b));
}
static std::vector<bf16> randomRows(size_t n, uint32_t seed) {
  std::mt19937 rng(seed);
  std::vector<bf16> v(n);
  for (auto &x : v)
    x = (bf16)(2.f * (float)(rng() >> 8) * (1.f / 16777216.f) - 1.f);
  return v;
}
static std::vector<float> floats(const std::shared_ptr<Buffer> &b) {
  std::vector<bf16> x;
  auto st = b->read(gpu(), x);
  if (isError(st))
    std::printf("read failed: %s\n", st.getMessage().c_str());
  return std::vector<float>(x.begin(), x.end());
}

TEST("a prompt, a chunk behind it and single tokens through graphs that share a cache") {
  const std::vector<int32_t> table = {3, 7, 1, 10, 5, 0, 11, 2};
  const Dims pool = {kPool, kHk, kPage, kD};
  auto cacheK = bufOf(std::vector<bf16>(kPool * kHk * kPage * kD, (bf16)0.f), pool);
  auto cacheV = bufOf(std::vector<bf16>(kPool * kHk * kPage * kD, (bf16)0.f), pool);
  std::vector<float> angles(kPlaces * kD);
  for (int64_t p = 0; p < kPlaces; ++p)
    for (int64_t i = 0; i < kD / 2; ++i) {
      const double a = p * std::pow(10000.0, -2.0 * i / kD);
      angles[p * kD + i] = (float)std::cos(a);
      angles[p * kD + kD / 2 + i] = (float)std::sin(a);
    }
  // what the cache has to hold, in double: [sequence][place][head][dim]
  std::vector<std::vector<double>> k(kBatch), v(kBatch);
  std::vector<int32_t> have(kBatch, 0);
  uint32_t seed = 1;
  const std::vector<std::vector<int32_t>> news = {{20, 3}, {7, 25}, {1, 1}, {1, 1}};
  for (size_t step = 0; step < news.size(); ++step) {
    const auto &n = news[step];
    const int64_t t = n[0] + n[1];
    const std::vector<int32_t> offsets = {0, n[0], n[0] + n[1]};
    for (int b = 0; b < kBatch; ++b)
      have[b] += n[b];
    Graph g = newGraph("step_" + std::to_string(step));
    Rows r = rowsOf(g, t);
    CacheTensors c = cacheOf(g);
    CacheAppendAttr aa;
    auto [qo, ko] = g.cacheAppend(r.q, r.k, r.v, r.rotation, nullptr, r.offsets, c, aa);
    TensorPtr o, kv; // the chunk goes through the rows read back
    Pack pack;
    if (step == 0) {
      SdpaPackedAttr pa;
      pa.setIsCausal(true);
      o = g.sdpaPacked(qo, ko, r.v, r.offsets, nullptr, pa);
    } else if (step == 1) {
      kv = g.tensor(mk("kv_offsets", {kBatch + 1}, DataType::Int32));
      CacheReadAttr ra;
      auto rows = g.cacheRead(kv, c, ra);
      rows[0]->setDim({have[0] + have[1], kHk, kD});
      rows[1]->setDim({have[0] + have[1], kHk, kD});
      SdpaPackedAttr pa;
      pa.setIsCausal(true);
      o = g.sdpaPacked(qo, rows[0], rows[1], r.offsets, kv, pa);
      pack[kv] = bufOf(std::vector<int32_t>{0, have[0], have[0] + have[1]}, {kBatch + 1});
    } else {
      SdpaPagedAttr pa;
      o = g.sdpaPaged(qo, r.offsets, c, pa);
    }
    o->setOutput(true);
    REQUIRE_OK(g.validate());
    REQUIRE_OK(g.compile(gpu(), true));
    const auto q = randomRows(t * kHq * kD, seed++), kNew = randomRows(t * kHk * kD, seed++),
               vNew = randomRows(t * kHk * kD, seed++);
    pack[r.q] = bufOf(q, {t, kHq, kD});
    pack[r.k] = bufOf(kNew, {t, kHk, kD});
    pack[r.v] = bufOf(vNew, {t, kHk, kD});
    pack[r.offsets] = bufOf(offsets, {kBatch + 1});
    pack[r.rotation] = bufOf(angles, {kPlaces, kD});
    pack[c.k] = cacheK;
    pack[c.v] = cacheV;
    pack[c.pages] = bufOf(table, {kBatch, kTable});
    pack[c.lengths] = bufOf(have, {kBatch});
    pack[o] = bufOf(std::vector<bf16>(t * kHq * kD, (bf16)7.f), {t, kHq, kD});
    auto need = g.getWorkspaceSize();
    REQUIRE(!isError(need) && need->has_value());
    std::shared_ptr<Buffer> ws;
    if (**need)
      ws = std::make_shared<Buffer>(std::move(*Buffer::allocateRaw(gpu(), **need)));
    for (int rep = 0; rep < 2; ++rep) { // (appending the same rows again changes nothing)
      REQUIRE_OK(g.execute(gpu(), pack, ws));
    }
    const auto got = floats(pack[o]);
    auto turned = [&](const std::vector<bf16> &x, int64_t row, int64_t heads, int64_t h, int64_t place, int64_t e) {
      const int64_t half = kD / 2, i = e % half;
      const bf16 *at = &x[(row * heads + h) * kD];
      const double cs = angles[place * kD + i], sn = angles[place * kD + half + i];
      const double a = (double)(float)at[i], b = (double)(float)at[half + i];
      return (double)(float)(bf16)(float)(e < half ? a * cs - b * sn : b * cs + a * sn);
    };
    for (int b = 0; b < kBatch; ++b)
      for (int i = 0; i < n[b]; ++i)
        for (int64_t h = 0; h < kHk; ++h)
          for (int64_t e = 0; e < kD; ++e) {
            const int64_t row = offsets[b] + i, place = have[b] - n[b] + i;
            k[b].resize((place + 1) * kHk * kD);
            v[b].resize((place + 1) * kHk * kD);
            k[b][(place * kHk + h) * kD + e] = turned(kNew, row, kHk, h, place, e);
            v[b][(place * kHk + h) * kD + e] = (double)(float)vNew[(row * kHk + h) * kD + e];
          }
    double worst = 0;
    for (int b = 0; b < kBatch; ++b)
      for (int i = 0; i < n[b]; ++i)
        for (int64_t h = 0; h < kHq; ++h) {
          const int64_t row = offsets[b] + i, place = have[b] - n[b] + i, hk = h / (kHq / kHk);
          std::vector<double> p(place + 1);
          double top = -1e300, sum = 0;
          for (int64_t j = 0; j <= place; ++j) {
            double s = 0;
            for (int64_t e = 0; e < kD; ++e)
              s += turned(q, row, kHq, h, place, e) * k[b][(j * kHk + hk) * kD + e];
            p[j] = s / std::sqrt((double)kD);
            top = std::max(top, p[j]);
          }
          for (double &x : p)
            sum += x = std::exp(x - top);
          for (int64_t e = 0; e < kD; ++e) {
            double ref = 0, size = 0;
            for (int64_t j = 0; j <= place; ++j) {
              ref += p[j] * v[b][(j * kHk + hk) * kD + e] / sum;
              size += p[j] * std::fabs(v[b][(j * kHk + hk) * kD + e]) / sum;
            }
            // probabilities and the result are rounded to bf16 (2^-8 each); a turned element that f32 and double round
            // apart moves a score by 2^-8 of one of 64 products of at most 2, an eighth of that behind the scale
            const double far = (size + std::fabs(ref)) / 256 * 1.02 + size * 2 * 2.0 / 256 / 8;
            worst = std::max(worst, std::fabs(got[(row * kHq + h) * kD + e] - ref) / far);
          }
        }
    std::printf("  step %zu: worst error %.3f of its bound\n", step, worst);
    CHECK(worst <= 1.0);
  }
}

TEST("buffers that give dynamic dims extents which do not belong together are refused") {
  Graph g = newGraph("dynamic");
  auto q = g.tensor(mk("q", {2, kHq, kD}, DataType::BFloat16));
  auto offsets = g.tensor(mk("offsets", {kBatch + 1}, DataType::Int32).setDynamicDims({0}));
  CacheTensors c = cacheOf(g);
  c.lengths->setDynamicDims({0});
  c.pages->setDynamicDims({0, 1});
  SdpaPagedAttr a;
  a.setName("p");
  auto o = g.sdpaPaged(q, offsets, c, a);
  o->setOutput(true);
  REQUIRE_OK(g.validate());
  REQUIRE_OK(g.compile(gpu(), true));
  auto need = g.getWorkspaceSize();
  REQUIRE(!isError(need) && **need == 0);
  const Dims pool = {kPool, kHk, kPage, kD};
  const std::vector<bf16> rows(kPool * kHk * kPage * kD, (bf16)1.f);
  auto run = [&](int64_t batch, int64_t table, int64_t nOffsets, int64_t nLengths) {
    Pack pack;
    pack[q] = bufOf(std::vector<bf16>(2 * kHq * kD, (bf16)1.f), {2, kHq, kD});
    pack[o] = bufOf(std::vector<bf16>(2 * kHq * kD, (bf16)7.f), {2, kHq, kD});
    pack[c.k] = bufOf(rows, pool);
    pack[c.v] = bufOf(rows, pool);
    pack[c.pages] = bufOf(std::vector<int32_t>(batch * table, 1), {batch, table});
    pack[c.lengths] = bufOf(std::vector<int32_t>(nLengths, 20), {nLengths});
    std::vector<int32_t> at(nOffsets, 2);
    at[0] = 0;
    pack[offsets] = bufOf(at, {nOffsets});
    auto st = g.execute(gpu(), pack, nullptr);
    if (!st.isError())
      for (float x : floats(pack[o]))
        CHECK(x == 1.f);
    return st;
  };
  REQUIRE_OK(run(2, 4, 3, 2));
  REQUIRE_OK(run(1, 3, 2, 1)); // both rows to one sequence
  CHECK_ERROR(run(2, 4, 2, 2), ErrorCode::InvalidAttribute, "Node 'p': tensor OFFSETS must be contiguous [3]");
  CHECK_ERROR(run(2, 4, 3, 1), ErrorCode::InvalidAttribute, "Node 'p': tensor LENGTHS must be contiguous [2]");
  CHECK_ERROR(run(1, 4, 3, 2), ErrorCode::InvalidAttribute, "Node 'p': tensor OFFSETS must be contiguous [2]");
}

int main(int argc, char **argv) { return mini::run(argc, argv); }
