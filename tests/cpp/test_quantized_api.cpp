// Models served in 8 bits through the graph API.  "host" cases need no GPU: what the nodes check, what a plan holds.
// The others run a layer, a head and the draw of tokens through one graph against plain loops in double.
#include <fusilli.h>

#include <algorithm>
#include <cmath>
#include <numeric>
#include <random>

#include "mini_test.h"

using namespace fusilli;
using Dims = std::vector<int64_t>;
using Pack = std::unordered_map<std::shared_ptr<TensorAttr>, std::shared_ptr<Buffer>>;
using Front = QuantizeRowsAttr::Front;

static Dims contig(const Dims &d) {
  return generateStrideFromDim(d, getContiguousStrideOrder(d.size()));
}
static TensorAttr mk(const std::string &name, Dims dim, DataType dt) {
  return TensorAttr().setName(name).setDim(dim).setStride(contig(dim)).setDataType(dt);
}
static Graph newGraph(const std::string &name) {
  Graph g;
  g.setName(name).setIODataType(DataType::BFloat16).setIntermediateDataType(DataType::Float)
      .setComputeDataType(DataType::Float);
  return g;
}

constexpr int64_t kRows = 6, kK = 192, kN = 320, kWords = 700;

TEST("host: quantizeRows checks its tensors") {
  struct Parts {
    TensorPtr x, up, weight, eps;
    Front front = Front::RMSNORM;
  };
  auto run = [](auto &&change) {
    Graph g = newGraph("quantize");
    Parts p;
    p.x = g.tensor(mk("x", {kRows, kK}, DataType::BFloat16));
    p.weight = g.tensor(mk("w", {1, kK}, DataType::BFloat16));
    p.eps = g.tensor(TensorAttr(1e-6f));
    change(g, p);
    QuantizeRowsAttr a;
    a.setName("q").setFront(p.front);
    if (p.eps)
      a.setEpsilon(p.eps);
    auto [q, s] = g.quantizeRows(p.x, p.up, p.weight, a);
    q->setOutput(true);
    s->setOutput(true);
    auto st = g.validate();
    if (!st.isError()) {
      CHECK(q->getDataType() == DataType::Int8 && s->getDataType() == DataType::Float);
      CHECK(q->getDim() == (Dims{kRows, kK}) && s->getDim() == (Dims{kRows, 1}));
    }
    return st;
  };
  REQUIRE_OK(run([](Graph &, Parts &) {}));
  CHECK_ERROR(run([](Graph &, Parts &p) { p.x = nullptr; }), ErrorCode::AttributeNotSet, "Quantize rows tensor X not set");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.x = g.tensor(mk("x3", {1, kRows, kK}, DataType::BFloat16)); }),
              ErrorCode::InvalidAttribute, "Quantize rows tensor X must be rank 2");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.weight = g.tensor(mk("w1", {1, kK + 1}, DataType::BFloat16)); }),
              ErrorCode::InvalidAttribute, "Quantize rows tensor WEIGHT must be [1, 192]");
  CHECK_ERROR(run([](Graph &, Parts &p) { p.eps = nullptr; }), ErrorCode::AttributeNotSet, "Quantize rows epsilon not set");
  CHECK_ERROR(run([](Graph &, Parts &p) { p.front = Front::NONE; }), ErrorCode::InvalidAttribute,
              "Quantize rows tensor WEIGHT needs the RMS norm");
  CHECK_ERROR(run([](Graph &, Parts &p) { p.front = Front::SWISH_GATE; }), ErrorCode::InvalidAttribute,
              "Quantize rows tensor UP and the swish gate go together");
}

TEST("host: matmulQuantized checks its tensors") {
  struct Parts {
    TensorPtr a, as, b, bs, bias;
  };
  auto run = [](auto &&change) {
    Graph g = newGraph("product");
    Parts p;
    p.a = g.tensor(mk("a", {kRows, kK}, DataType::Int8));
    p.b = g.tensor(mk("b", {kK, kN}, DataType::Int8));
    p.as = g.tensor(mk("as", {kRows, 1}, DataType::Float));
    p.bs = g.tensor(mk("bs", {1, kN}, DataType::Float));
    change(g, p);
    MatmulQuantizedAttr a;
    a.setName("m");
    g.matmulQuantized(p.a, p.as, p.b, p.bs, p.bias, a)->setOutput(true);
    return g.validate();
  };
  REQUIRE_OK(run([](Graph &, Parts &) {}));
  REQUIRE_OK(run([](Graph &g, Parts &p) { p.as = g.tensor(mk("one", {1, 1}, DataType::Float)); }));
  REQUIRE_OK(run([](Graph &g, Parts &p) { p.bias = g.tensor(mk("bias", {1, kN}, DataType::Half)); }));
  CHECK_ERROR(run([](Graph &, Parts &p) { p.bs = nullptr; }), ErrorCode::AttributeNotSet,
              "Quantized matmul tensors A_SCALE and B_SCALE must be set");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.b = g.tensor(mk("b1", {kK + 1, kN}, DataType::Int8)); }),
              ErrorCode::InvalidAttribute,
              "Quantized matmul input tensors A and B have incompatible inner dimensions (K): A has K=192, B has K=193");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.as = g.tensor(mk("as1", {kRows + 1, 1}, DataType::Float)); }),
              ErrorCode::InvalidAttribute, "Quantized matmul tensor A_SCALE must be [6, 1] or [1, 1]");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.bs = g.tensor(mk("bs16", {1, kN}, DataType::BFloat16)); }),
              ErrorCode::InvalidAttribute, "Quantized matmul tensor B_SCALE must be Float");
  CHECK_ERROR(run([](Graph &g, Parts &p) { p.bias = g.tensor(mk("bias1", {kN, 1}, DataType::Float)); }),
              ErrorCode::InvalidAttribute, "Quantized matmul tensor BIAS must be [1, 320] or [1, 1]");
}

TEST("host: sample checks its tensors") {
  auto run = [](auto &&change) {
    Graph g = newGraph("sample");
    TensorPtr in[6] = {g.tensor(mk("logits", {kRows, kWords}, DataType::Float)), g.tensor(mk("u", {kRows}, DataType::Float))};
    change(g, in);
    SampleAttr a;
    a.setName("s");
    auto [token, probability] = g.sample(in[0], in[1], in[2], in[3], in[4], in[5], a);
    token->setOutput(true);
    auto st = g.validate();
    if (!st.isError())
      CHECK(token->getDataType() == DataType::Int32 && token->getDim() == (Dims{kRows}));
    return st;
  };
  REQUIRE_OK(run([](Graph &, TensorPtr *) {}));
  REQUIRE_OK(run([](Graph &g, TensorPtr *in) {
    in[2] = g.tensor(TensorAttr(0.7f));
    in[3] = g.tensor(TensorAttr(int64_t{1} << 40));
    in[4] = g.tensor(mk("p", {kRows}, DataType::Float));
  }));
  CHECK_ERROR(run([](Graph &, TensorPtr *in) { in[1] = nullptr; }), ErrorCode::AttributeNotSet, "Sample tensor UNIFORM not set");
  CHECK_ERROR(run([](Graph &g, TensorPtr *in) { in[1] = g.tensor(TensorAttr(0.5f)); }), ErrorCode::InvalidAttribute,
              "Sample tensor UNIFORM must not be a constant");
  CHECK_ERROR(run([](Graph &g, TensorPtr *in) { in[3] = g.tensor(mk("k", {kRows}, DataType::Float)); }),
              ErrorCode::InvalidAttribute, "Sample tensor TOP_K must be Int32");
  CHECK_ERROR(run([](Graph &g, TensorPtr *in) { in[5] = g.tensor(mk("m", {kRows + 1}, DataType::Float)); }),
              ErrorCode::InvalidAttribute, "Sample tensor MIN_P must be contiguous [6]");
  CHECK_ERROR(run([](Graph &g, TensorPtr *in) { in[0] = g.tensor(mk("l1", {kWords}, DataType::Float)); }),
              ErrorCode::InvalidAttribute, "Sample tensor LOGITS must be rank 2");
}

struct Layer {
  TensorPtr x, weight, b1, bs1, rest, b2, bs2, u, t, p;
  TensorPtr q1, s1, hidden, q2, s2, logits, token, probability;
};
// norm and codes, a product with GELU and a residual, codes, the head's product, tokens
static Layer layerOf(Graph &g) {
  Layer l;
  l.x = g.tensor(mk("x", {kRows, kK}, DataType::BFloat16));
  l.weight = g.tensor(mk("weight", {1, kK}, DataType::BFloat16));
  l.b1 = g.tensor(TensorAttr().setName("b1").setDim({kK, kN}).setStride({1, kK}).setDataType(DataType::Int8));
  l.bs1 = g.tensor(mk("bs1", {1, kN}, DataType::Float));
  l.rest = g.tensor(mk("rest", {kRows, kN}, DataType::BFloat16));
  l.b2 = g.tensor(TensorAttr().setName("b2").setDim({kN, kWords}).setStride({1, kN}).setDataType(DataType::Int8));
  l.bs2 = g.tensor(mk("bs2", {1, kWords}, DataType::Float));
  l.u = g.tensor(mk("u", {kRows}, DataType::Float));
  l.t = g.tensor(mk("t", {kRows}, DataType::Float));
  l.p = g.tensor(TensorAttr(0.9f));
  QuantizeRowsAttr q1;
  q1.setName("q1").setFront(Front::RMSNORM).setEpsilon(g.tensor(TensorAttr(1e-6f)));
  auto first = g.quantizeRows(l.x, nullptr, l.weight, q1);
  l.q1 = first[0], l.s1 = first[1];
  MatmulQuantizedAttr m1;
  m1.setName("m1");
  auto c = g.matmulQuantized(l.q1, l.s1, l.b1, l.bs1, nullptr, m1);
  PointwiseAttr gelu, add;
  gelu.setName("gelu").setMode(PointwiseAttr::Mode::GELU_FWD);
  add.setName("add").setMode(PointwiseAttr::Mode::ADD);
  l.hidden = g.pointwise(g.pointwise(c, gelu), l.rest, add);
  QuantizeRowsAttr q2;
  q2.setName("q2");
  auto second = g.quantizeRows(l.hidden, nullptr, nullptr, q2);
  l.q2 = second[0], l.s2 = second[1];
  MatmulQuantizedAttr m2;
  m2.setName("m2");
  l.logits = g.matmulQuantized(l.q2, l.s2, l.b2, l.bs2, nullptr, m2);
  SampleAttr sa;
  sa.setName("s");
  auto drawn = g.sample(l.logits, l.u, l.t, nullptr, l.p, nullptr, sa);
  l.token = drawn[0], l.probability = drawn[1];
  return l;
}

TEST("host: a layer, a head and a draw are five kernels; what is between them lies in the workspace") {
  Graph g = newGraph("layer");
  Layer l = layerOf(g);
  l.hidden->setDataType(DataType::BFloat16);
  l.token->setOutput(true);
  REQUIRE_OK(g.validate());
  REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
  REQUIRE_OK(g.compile(cpu, true));
  CHECK(g.getKernelCount() == std::optional<size_t>(5));
  auto ws = g.getWorkspaceSize();
  REQUIRE(!isError(ws) && ws->has_value());
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int64_t between = up(kRows * kK) + up(kRows * 4) + up(kRows * kN * 2) + up(kRows * kN) + up(kRows * 4) + up(kRows * kWords * 4);
  CHECK(**ws >= between); // (and what the draw needs; an unread PROBABILITY has no place)
  CHECK(l.probability->isVirtual());
}

TEST("host: what no kernel takes is refused by compile") {
  Graph g = newGraph("refused");
  MatmulQuantizedAttr a;
  a.setName("m");
  g.matmulQuantized(g.tensor(mk("a", {kRows, kK}, DataType::Uint8)), g.tensor(mk("as", {kRows, 1}, DataType::Float)),
                    g.tensor(mk("b", {kK, kN}, DataType::Int8)), g.tensor(mk("bs", {1, kN}, DataType::Float)), nullptr, a)
      ->setOutput(true);
  REQUIRE_OK(g.validate());
  REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
  CHECK_ERROR(g.compile(cpu, true), ErrorCode::NotImplemented,
              "Quantized matmul node 'm' is not executable by this backend: fhip_matmul_quantized: A and B must be Int8");
}

TEST("host: buffers give a draw another number of rows, also where nothing asks for the probability") {
  for (bool asked : {false, true}) {
    Graph g = newGraph("dynamic_draw");
    auto logits = g.tensor(mk("logits", {kRows, kWords}, DataType::Float).setDynamicDims({0}));
    auto u = g.tensor(mk("u", {kRows}, DataType::Float).setDynamicDims({0}));
    SampleAttr a;
    a.setName("s");
    auto [token, probability] = g.sample(logits, u, g.tensor(TensorAttr(0.8f)), nullptr, nullptr, nullptr, a);
    token->setOutput(true).setDim({kRows}).setStride({1}).setDynamicDims({0});
    if (asked)
      probability->setOutput(true).setDim({kRows}).setStride({1}).setDynamicDims({0});
    REQUIRE_OK(g.validate());
    REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
    REQUIRE_OK(g.compile(cpu, true));
    auto need = g.getWorkspaceSize();
    REQUIRE(!isError(need) && **need == 0);
    for (int64_t rows : {kRows, int64_t{1}, int64_t{50}}) {
      auto buf = [&](int64_t cols, const Dims &dims) {
        return std::make_shared<Buffer>(std::move(*Buffer::allocate(
            cpu, std::vector<size_t>(dims.begin(), dims.end()), std::vector<float>(rows * cols))));
      };
      Pack pack;
      pack[logits] = buf(kWords, {rows, kWords});
      pack[u] = buf(1, {rows});
      pack[token] = std::make_shared<Buffer>(
          std::move(*Buffer::allocate(cpu, {(size_t)rows}, std::vector<int32_t>(rows))));
      if (asked)
        pack[probability] = buf(1, {rows});
      // (planned for these rows: only then the backend is looked at)
      CHECK_ERROR(g.execute(cpu, pack, nullptr), ErrorCode::NotImplemented,
                  "Backend::CPU has no execution engine in this build: graphs run on Backend::AMDGPU (gfx950) only");
      if (asked && rows != kRows) {
        pack[probability] = std::make_shared<Buffer>(
            std::move(*Buffer::allocate(cpu, {(size_t)kRows}, std::vector<float>(kRows))));
        CHECK_ERROR(g.execute(cpu, pack, nullptr), ErrorCode::InvalidAttribute,
                    "Node 's': tensor PROBABILITY must be contiguous [" + std::to_string(rows) + "]");
      }
    }
  }
}

TEST("host: the workspace of a draw with dynamic rows serves every number of rows up to the declared one") {
  constexpr int64_t kLong = 30000;
  auto needOf = [&](int64_t rows, bool dynamic) {
    Graph g = newGraph("dynamic_room");
    auto logits = g.tensor(mk("logits", {rows, kLong}, DataType::Half));
    auto u = g.tensor(mk("u", {rows}, DataType::Float));
    SampleAttr a;
    a.setName("s");
    auto token = g.sample(logits, u, nullptr, nullptr, nullptr, nullptr, a)[0];
    token->setOutput(true);
    if (dynamic) {
      logits->setDynamicDims({0});
      u->setDynamicDims({0});
      token->setDim({rows}).setStride({1}).setDynamicDims({0});
    }
    REQUIRE_OK(g.validate());
    REQUIRE_ASSIGN(Handle cpu, Handle::create(Backend::CPU));
    REQUIRE_OK(g.compile(cpu, true));
    auto need = g.getWorkspaceSize();
    REQUIRE(!isError(need) && need->has_value());
    return **need;
  };
  // (few long rows are cut into parts, many are not)
  CHECK(needOf(256, false) == 0);
  for (int64_t rows : {2, 100, 256, 1000}) {
    const size_t room = needOf(rows, true);
    for (int64_t now : {1, 2, 5, 60, 127, 128, 190, 191, 192, 256})
      if (now <= rows)
        CHECK(room >= needOf(now, false));
  }
}

TEST("host: constants of TOP_K that are no count are off, larger ones all words") {
  auto planOf = [](float k) {
    Graph g = newGraph("constant_top_k");
    auto logits = g.tensor(mk("logits", {kRows, kWords}, DataType::Float));
    SampleAttr a;
    a.setName("s");
    g.sample(logits, g.tensor(mk("u", {kRows}, DataType::Float)), nullptr, g.tensor(TensorAttr(k)), nullptr, nullptr, a)[0]
        ->setOutput(true);
    REQUIRE_OK(g.validate());
    REQUIRE_ASSIGN(auto bytes, g.compileToArtifact(Backend::CPU, /*remove=*/true));
    return bytes;
  };
  const auto off = planOf(0.f), all = planOf(2147483648.f);
  CHECK(off != all && off != planOf(1.f));
  for (float k : {std::nanf(""), -1.f, 0.5f, -INFINITY})
    CHECK(planOf(k) == off);
  for (float k : {1e30f, INFINITY})
    CHECK(planOf(k) == all);
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
template <typename T> static std::vector<T> read(const std::shared_ptr<Buffer> &b) {
  std::vector<T> x;
  auto st = b->read(gpu(), x);
  if (isError(st))
    std::printf("read failed: %s\n", st.getMessage().c_str());
  return x;
}

TEST("a layer, a head and a draw through one graph") {
  Graph g = newGraph("layer_gpu");
  Layer l = layerOf(g);
  l.hidden->setDataType(DataType::BFloat16);
  for (const auto &t : {l.q1, l.s1, l.hidden, l.q2, l.s2, l.logits, l.token, l.probability})
    t->setOutput(true);
  l.logits->setDataType(DataType::Float);
  REQUIRE_OK(g.validate());
  REQUIRE_OK(g.compile(gpu(), true));
  CHECK(g.getKernelCount() == std::optional<size_t>(5));
  std::mt19937 rng(7);
  std::normal_distribution<float> normal;
  std::uniform_real_distribution<float> even(0.f, 1.f);
  auto rows = [&](size_t n, float by, float plus) {
    std::vector<bf16> v(n);
    for (auto &x : v)
      x = (bf16)(normal(rng) * by + plus);
    return v;
  };
  auto codes = [&](size_t n) {
    std::vector<int8_t> v(n);
    for (auto &x : v)
      x = (int8_t)std::clamp(std::nearbyint(normal(rng) * 40.f), -127.f, 127.f);
    return v;
  };
  auto scales = [&](size_t n, float by) {
    std::vector<float> v(n);
    for (auto &x : v)
      x = by * (0.5f + even(rng));
    return v;
  };
  const auto x = rows(kRows * kK, 1.f, 0.f), weight = rows(kK, 0.1f, 1.f), rest = rows(kRows * kN, 1.f, 0.f);
  const auto b1 = codes(kK * kN), b2 = codes(kN * kWords);
  const auto bs1 = scales(kN, 0.002f), bs2 = scales(kWords, 0.004f), u = scales(kRows, 0.6f), t = scales(kRows, 1.f);
  Pack pack;
  pack[l.x] = bufOf(x, {kRows, kK});
  pack[l.weight] = bufOf(weight, {1, kK});
  pack[l.rest] = bufOf(rest, {kRows, kN});
  pack[l.b1] = bufOf(b1, {kK, kN});
  pack[l.b2] = bufOf(b2, {kN, kWords});
  pack[l.bs1] = bufOf(bs1, {1, kN});
  pack[l.bs2] = bufOf(bs2, {1, kWords});
  pack[l.u] = bufOf(u, {kRows});
  pack[l.t] = bufOf(t, {kRows});
  pack[l.q1] = bufOf(std::vector<int8_t>(kRows * kK, 99), {kRows, kK});
  pack[l.q2] = bufOf(std::vector<int8_t>(kRows * kN, 99), {kRows, kN});
  pack[l.s1] = bufOf(std::vector<float>(kRows, 9.f), {kRows, 1});
  pack[l.s2] = bufOf(std::vector<float>(kRows, 9.f), {kRows, 1});
  pack[l.hidden] = bufOf(std::vector<bf16>(kRows * kN, (bf16)9.f), {kRows, kN});
  pack[l.logits] = bufOf(std::vector<float>(kRows * kWords, 9.f), {kRows, kWords});
  pack[l.token] = bufOf(std::vector<int32_t>(kRows, 9), {kRows});
  pack[l.probability] = bufOf(std::vector<float>(kRows, 9.f), {kRows});
  auto need = g.getWorkspaceSize();
  REQUIRE(!isError(need) && need->has_value());
  std::shared_ptr<Buffer> ws;
  if (**need)
    ws = std::make_shared<Buffer>(std::move(*Buffer::allocateRaw(gpu(), **need)));
  for (int rep = 0; rep < 2; ++rep)
    REQUIRE_OK(g.execute(gpu(), pack, ws));
  const auto q1 = read<int8_t>(pack[l.q1]), q2 = read<int8_t>(pack[l.q2]);
  const auto s1 = read<float>(pack[l.s1]), s2 = read<float>(pack[l.s2]), logits = read<float>(pack[l.logits]),
             probability = read<float>(pack[l.probability]);
  const auto hidden = read<bf16>(pack[l.hidden]);
  const auto token = read<int32_t>(pack[l.token]);
  const double unit = std::ldexp(1.0, -24);
  for (int64_t r = 0; r < kRows; ++r) {
    // codes of the norm, off by the f32 steps of y (a sum of 192 squares, six roundings) and half a code
    auto codesOf = [&](const std::vector<double> &y, const int8_t *q, float s, double rel) {
      double most = 0;
      for (double v : y)
        most = std::max(most, std::fabs(v));
      CHECK(std::fabs(s - most / 127) <= (rel + unit) * most / 127);
      bool fine = true;
      for (size_t k = 0; k < y.size(); ++k)
        fine = fine && std::fabs(q[k] - y[k] * 127 / most) <= 0.5 + 127 * 2 * (rel + unit);
      CHECK(fine);
    };
    double sum = 0;
    std::vector<double> y(kK), h(kN);
    for (int64_t k = 0; k < kK; ++k)
      sum += (double)(float)x[r * kK + k] * (double)(float)x[r * kK + k];
    for (int64_t k = 0; k < kK; ++k)
      y[k] = (double)(float)x[r * kK + k] / std::sqrt(sum / kK + 1e-6) * (double)(float)weight[k];
    codesOf(y, &q1[r * kK], s1[r], 14 * unit);
    bool fine = true;
    for (int64_t n = 0; n < kN; ++n) {
      int64_t dot = 0;
      for (int64_t k = 0; k < kK; ++k)
        dot += (int64_t)q1[r * kK + k] * b1[n * kK + k];
      const double c = (double)dot * s1[r] * bs1[n], add = (double)(float)rest[r * kN + n];
      const double gelu = 0.5 * c * (1 + std::erf(c / std::sqrt(2.0)));
      // three roundings of c, GELU's kernel (2e-6 of it and 4e-7), the sum, bf16
      const double far = 3 * unit * std::fabs(c) * 1.2 + 2e-6 * std::fabs(gelu) + 4e-7 + (unit + 1.0 / 256) * std::fabs(gelu + add);
      h[n] = (double)(float)hidden[r * kN + n];
      fine = fine && std::fabs(h[n] - gelu - add) <= far;
    }
    CHECK(fine);
    codesOf(h, &q2[r * kN], s2[r], 0.0);
    fine = true;
    for (int64_t n = 0; n < kWords; ++n) {
      int64_t dot = 0;
      for (int64_t k = 0; k < kN; ++k)
        dot += (int64_t)q2[r * kN + k] * b2[n * kN + k];
      const double c = (double)dot * s2[r] * bs2[n];
      fine = fine && std::fabs(logits[r * kWords + n] - c) <= 4 * unit * std::fabs(c);
    }
    CHECK(fine);
    std::vector<int> order(kWords);
    std::iota(order.begin(), order.end(), 0);
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return logits[r * kWords + a] > logits[r * kWords + b]; });
    std::vector<double> w(kWords);
    for (int64_t n = 0; n < kWords; ++n)
      w[n] = std::exp(((double)logits[r * kWords + order[n]] - (double)logits[r * kWords + order[0]]) / t[r]);
    const double share = (double)0.9f * std::accumulate(w.begin(), w.end(), 0.0);
    double kept = 0, run = 0;
    int64_t count = 0;
    while (count < kWords && kept < share)
      kept += w[count++];
    int64_t at = 0;
    while (at < count - 1 && (run += w[at]) <= (double)u[r] * kept)
      ++at;
    CHECK(token[r] == order[at]);
    CHECK(std::fabs(probability[r] - w[at] / kept) <= 1e-6 * w[at] / kept);
  }
}

TEST("buffers that give dynamic dims extents which do not belong together are refused") {
  Graph g = newGraph("dynamic");
  auto a = g.tensor(mk("a", {kRows, kK}, DataType::Int8).setDynamicDims({0}));
  auto as = g.tensor(mk("as", {kRows, 1}, DataType::Float).setDynamicDims({0}));
  auto b = g.tensor(mk("b", {kK, kN}, DataType::Int8));
  auto bs = g.tensor(mk("bs", {1, kN}, DataType::Float));
  MatmulQuantizedAttr attr;
  attr.setName("m");
  auto c = g.matmulQuantized(a, as, b, bs, nullptr, attr);
  c->setOutput(true).setDataType(DataType::Float).setDim({kRows, kN}).setStride({kN, 1}).setDynamicDims({0});
  REQUIRE_OK(g.validate());
  REQUIRE_OK(g.compile(gpu(), true));
  auto need = g.getWorkspaceSize();
  REQUIRE(!isError(need) && **need == 0);
  auto run = [&](int64_t rows, int64_t nScales) {
    Pack pack;
    pack[a] = bufOf(std::vector<int8_t>(rows * kK, 2), {rows, kK});
    pack[b] = bufOf(std::vector<int8_t>(kK * kN, 3), {kK, kN});
    pack[as] = bufOf(std::vector<float>(nScales, 0.5f), {nScales, 1});
    pack[bs] = bufOf(std::vector<float>(kN, 0.25f), {1, kN});
    pack[c] = bufOf(std::vector<float>(rows * kN, 7.f), {rows, kN});
    auto st = g.execute(gpu(), pack, nullptr);
    if (!st.isError())
      for (float x : read<float>(pack[c]))
        CHECK(x == 0.125f * 6 * kK);
    return st;
  };
  REQUIRE_OK(run(kRows, kRows));
  REQUIRE_OK(run(3, 3));
  REQUIRE_OK(run(200, 200));
  CHECK_ERROR(run(5, 4), ErrorCode::InvalidAttribute, "Node 'm': tensor A_SCALE must be [5, 1] or [1, 1]");
}

int main(int argc, char **argv) { return mini::run(argc, argv); }
