// TextGenerator::GenerateBatch over a toy model: hidden states are a fixed function of
// the context, and all numbers are small whole ones, so that the head's sums are exact
// and a request's tokens can be compared with those of the request alone and with the
// host's own arithmetic. `--refusals-only` runs what needs no GPU.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include <cuda_fp16.h>

#include "neuraval_generation.hpp"

using namespace neuraval;

static int g_fail = 0, g_run = 0;
#define EXPECT(cond, what)                                                     \
  do {                                                                         \
    ++g_run;                                                                   \
    if (!(cond)) {                                                             \
      ++g_fail;                                                                \
      std::fprintf(stderr, "FAIL %s: %s\n", std::string(what).c_str(), #cond); \
    }                                                                          \
  } while (0)
template <typename E, typename F>
static bool throws(F f) {
  try {
    f();
  } catch (const E&) {
    return true;
  } catch (...) {
  }
  return false;
}

static uint64_t mix(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
static int small(uint64_t seed) { return static_cast<int>(mix(seed * 0x9E3779B97F4A7C15ull) % 5) - 2; }

constexpr int IN = 96, V = 1500, RANK = 4, SLOTS = 2;
static std::vector<int> hidden_of(const std::vector<int>& ctx) {
  uint64_t h = 1469598103934665603ull;
  for (int t : ctx) h = (h ^ static_cast<uint64_t>(static_cast<uint32_t>(t))) * 1099511628211ull;
  std::vector<int> x(IN);
  for (int i = 0; i < IN; ++i) x[i] = small(h + i);
  return x;
}
static int weight(int v, int i) { return small(1000003ull * v + i + 17); }
static int mat_a(int s, int r, int i) { return small(7777777ull * (s + 1) + 131 * r + i); }
static int mat_b(int s, int v, int r) { return small(5555557ull * (s + 1) + 13 * v + r); }
static std::vector<double> logits_of(const std::vector<int>& ctx, int slot) {
  const std::vector<int> x = hidden_of(ctx);
  std::vector<double> y(V);
  int u[RANK] = {};
  if (slot >= 0)
    for (int r = 0; r < RANK; ++r)
      for (int i = 0; i < IN; ++i) u[r] += mat_a(slot, r, i) * x[i];
  for (int v = 0; v < V; ++v) {
    int sum = 0;
    for (int i = 0; i < IN; ++i) sum += weight(v, i) * x[i];
    y[v] = sum / 8.0;
    for (int r = 0; r < RANK && slot >= 0; ++r) y[v] += 0.25 * u[r] * mat_b(slot, v, r) / 8.0;
  }
  return y;
}

struct Buffer {
  void* p = nullptr;
  explicit Buffer(size_t bytes) {
    if (cudaMalloc(&p, bytes) != cudaSuccess) throw CudaException(NCB_ERROR_ALLOC_FAILED, "cudaMalloc");
  }
  ~Buffer() { cudaFree(p); }
  void fill(const std::vector<__half>& h) { cudaMemcpy(p, h.data(), h.size() * 2, cudaMemcpyHostToDevice); }
};

static void batch_tests() {
  Device dev(0, 1, V, 16);
  cudaStream_t st = nullptr;
  cudaStreamCreate(&st);
  {
    AdapterHead head(0, NCB_DTYPE_F16, IN, V, 8, SLOTS, RANK);
    Buffer w(2 * V * IN), a(2 * RANK * IN), b(2 * V * RANK), x(2 * 8 * IN);
    std::vector<__half> host(V * IN);
    for (int v = 0; v < V; ++v)
      for (int i = 0; i < IN; ++i) host[v * IN + i] = __float2half(weight(v, i) / 8.0f);
    w.fill(host);
    head.SetWeight(w.p, IN, st);
    for (int s = 0; s < SLOTS; ++s) {
      host.assign(RANK * IN, __float2half(0));
      for (int r = 0; r < RANK; ++r)
        for (int i = 0; i < IN; ++i) host[r * IN + i] = __float2half(static_cast<float>(mat_a(s, r, i)));
      a.fill(host);
      host.assign(V * RANK, __float2half(0));
      for (int v = 0; v < V; ++v)
        for (int r = 0; r < RANK; ++r) host[v * RANK + r] = __float2half(mat_b(s, v, r) / 8.0f);
      b.fill(host);
      head.SetAdapter(s, a.p, IN, b.p, RANK, RANK, 0.25f, st);
      cudaStreamSynchronize(st);
    }
    int calls = 0;
    size_t longest = 0;
    const TextGenerator::HiddenModel model = [&](const std::vector<std::vector<int>>& contexts,
                                                 cudaStream_t stream) {
      ++calls;
      std::vector<__half> rows;
      for (const auto& c : contexts) {
        longest = std::max(longest, c.size());
        for (int v : hidden_of(c)) rows.push_back(__float2half(static_cast<float>(v)));
      }
      cudaMemcpyAsync(x.p, rows.data(), rows.size() * 2, cudaMemcpyHostToDevice, stream);
      cudaStreamSynchronize(stream);  // rows is a temporary
      return static_cast<const void*>(x.p);
    };
    const std::vector<int> none;
    TextGenerator gen(dev, 12);
    std::vector<BatchRequest> rq;
    rq.push_back({{3, 1, 4}, GenerationOptions::CreateGreedy(20, none), 0.0f, 0});
    rq.push_back({{1, 5}, GenerationOptions::Create(false, 0.9f, 0.9f, 40, 1.0f, 9, none, 11), 0.05f, 1});
    rq.push_back({{9}, GenerationOptions::Create(false, 1.3f, 0.8f, INT_MAX, 1.0f, 30, none, 12), 0.0f, -1});
    rq.push_back({{2, 6, 5}, GenerationOptions::Create(false, 0.7f, 1.0f, 50, 1.0f, 25, none, 13), 0.2f, 0});
    rq.push_back({{3, 1, 4}, GenerationOptions::CreateGreedy(20, none), 0.0f, -1});
    const auto all = gen.GenerateBatch(model, head, rq, st);
    EXPECT(calls == 30 && longest == 12, "one call of the model a step, contexts within the window");
    bool alone = true;
    for (size_t i = 0; i < rq.size(); ++i) {
      EXPECT(all[i].GeneratedTokenIds.size() == static_cast<size_t>(rq[i].Options.MaxNewTokens()),
             "every request has its own length");
      alone = alone && gen.GenerateBatch(model, head, {rq[i]}, st)[0].GeneratedTokenIds ==
                           all[i].GeneratedTokenIds;
    }
    EXPECT(alone, "a request's tokens are those of the request alone");
    // greedy requests: the host's own argmax, with and without the adapter
    for (size_t i : {size_t{0}, size_t{4}}) {
      std::vector<int> seq = rq[i].PromptTokenIds;
      bool same = true;
      for (int t : all[i].GeneratedTokenIds) {
        const std::vector<int> ctx(seq.size() > 12 ? seq.end() - 12 : seq.begin(), seq.end());
        const std::vector<double> y = logits_of(ctx, rq[i].Adapter);
        same = same && t == static_cast<int>(std::max_element(y.begin(), y.end()) - y.begin());
        seq.push_back(t);
      }
      EXPECT(same, "greedy tokens are the first maximum of W x + scale B (A x)");
    }
    EXPECT(all[0].GeneratedTokenIds != all[4].GeneratedTokenIds, "the adapter changes what is said");
    // a stop token ends its request alone
    rq[3].Options = GenerationOptions::Create(false, 0.7f, 1.0f, 50, 1.0f, 25,
                                              std::vector<int>{all[3].GeneratedTokenIds[4]}, 13);
    const auto cut = gen.GenerateBatch(model, head, rq, st);
    EXPECT(cut[3].FinishReason == GenerationFinishReason::StopToken &&
               cut[3].GeneratedTokenIds.size() <= 5 && cut[2].GeneratedTokenIds == all[2].GeneratedTokenIds,
           "a stop token ends its request and no other");
    EXPECT(gen.GenerateBatch(model, head, {}, st).empty(), "no requests");
    // refusals
    auto bad = rq;
    bad[1].Options = GenerationOptions::Create(false, 0.9f, 0.9f, 40, 1.1f, 9, none);
    EXPECT(throws<ArgumentException>([&] { gen.GenerateBatch(model, head, bad, st); }), "penalty");
    bad = rq;
    bad[0].MinP = 1.5f;
    EXPECT(throws<ArgumentOutOfRangeException>([&] { gen.GenerateBatch(model, head, bad, st); }), "minP");
    bad = rq;
    bad[2].PromptTokenIds.clear();
    EXPECT(throws<ArgumentException>([&] { gen.GenerateBatch(model, head, bad, st); }), "prompt");
    bad = rq;
    while (bad.size() <= 8) bad.push_back(rq[0]);
    EXPECT(throws<ArgumentOutOfRangeException>([&] { gen.GenerateBatch(model, head, bad, st); }), "rows");
    EXPECT(throws<ArgumentException>([&] { gen.GenerateBatch(model, head, rq, st, {nullptr}); }), "randoms");
    EXPECT(throws<ArgumentNullException>([&] { gen.GenerateBatch(nullptr, head, rq, st); }), "model");
  }
  cudaStreamDestroy(st);
}

int main(int argc, char** argv) {
  EXPECT(throws<CudaException>([] { AdapterHead(0, NCB_DTYPE_F32, 8, 8, 1); }), "fp32 weights");
  EXPECT(throws<CudaException>([] { AdapterHead(0, NCB_DTYPE_F16, 8, 8, 1, 4, 0); }), "adapters of no rank");
  if (argc < 2 || std::strcmp(argv[1], "--refusals-only") != 0) batch_tests();
  std::printf("%d checks, %d failed\n", g_run, g_fail);
  return g_fail == 0 ? 0 : 1;
}
