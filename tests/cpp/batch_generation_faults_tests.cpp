// TextGenerator::GenerateBatch where something goes wrong for one request, or for all: the
// largest draws, rows without a token, a head whose kernel gave up. `--no-gpu` runs what
// needs no GPU.
#include <dlfcn.h>

#include <chrono>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <thread>
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

// Stands in for the library's: what the head's kernels are said to have come to.
static int g_status = NCB_OK;
extern "C" int ncb_adapter_head_status(NcbAdapterHead*) { return g_status; }

// And this one refuses when it is told to, behind work that takes its time.
static bool g_refuse = false, g_ended = false;
extern "C" int ncb_sample_rows_min_p_device(const void* logits, int dtype, int rows, int vocab, int64_t ld, const float* u,
                                            const float* T, const int32_t* k, const float* p, const float* m,
                                            int32_t* tokens, float* lp, int32_t* kept, uint32_t* flags, void* stream) {
  static const auto next = reinterpret_cast<decltype(&ncb_sample_rows_min_p_device)>(dlsym(RTLD_NEXT, "ncb_sample_rows_min_p_device"));
  if (!g_refuse) return next(logits, dtype, rows, vocab, ld, u, T, k, p, m, tokens, lp, kept, flags, stream);
  cudaLaunchHostFunc(static_cast<cudaStream_t>(stream), [](void*) {
    std::this_thread::sleep_for(std::chrono::milliseconds(50));
    g_ended = true;
  }, nullptr);
  return NCB_ERROR_CAPACITY;
}

struct Fixed final : Random {
  double u;
  explicit Fixed(double v) : u(v) {}
  double NextDouble() override { return u; }
};

static void draw_tests() {
  EXPECT(UniformBelowOne(0.0) == 0.0f && UniformBelowOne(0.3) == 0.3f, "ordinary draws as they are");
  for (double u : {1.0 - 0x1p-24, 1.0 - 0x1p-25, 1.0 - 0x1p-26, 1.0 - 0x1p-53})
    EXPECT(UniformBelowOne(u) == 1.0f - 0x1p-24f, "the largest draws stay below 1");
}

constexpr int IN = 32, V = 300, ROWS = 8;
static int small(uint64_t z) {
  z = z * 0x9E3779B97F4A7C15ull + 0x1234567ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  return static_cast<int>((z ^ (z >> 27)) % 5) - 2;
}
struct Buffer {
  void* p = nullptr;
  explicit Buffer(size_t bytes) {
    if (cudaMalloc(&p, bytes) != cudaSuccess) throw CudaException(NCB_ERROR_ALLOC_FAILED, "cudaMalloc");
  }
  ~Buffer() { cudaFree(p); }
  void fill(const std::vector<__half>& h) { cudaMemcpy(p, h.data(), h.size() * 2, cudaMemcpyHostToDevice); }
};

// A head with sound adapters in slot 0 and one with a NaN in slot 1, and a toy model whose
// hidden state is NaN for contexts that begin with `poisoned` and have `from` tokens or more.
struct Bench {
  cudaStream_t st = nullptr;
  Device dev{0, 1, V, 16};
  AdapterHead head{0, NCB_DTYPE_F16, IN, V, ROWS, 2, 4};
  Buffer w{2 * V * IN}, a{2 * 4 * IN}, b{2 * V * 4}, x{2 * ROWS * IN};
  TextGenerator gen{dev, 64};
  int poisoned = -1;
  size_t from = 0;
  Bench() {
    cudaStreamCreate(&st);
    std::vector<__half> h;
    for (int i = 0; i < V * IN; ++i) h.push_back(__float2half(small(i) / 8.0f));
    w.fill(h);
    head.SetWeight(w.p, IN, st);
    for (int slot = 0; slot < 2; ++slot) {
      h.clear();
      for (int i = 0; i < 4 * IN; ++i) h.push_back(__float2half(small(7000 + i) / 8.0f));
      a.fill(h);
      h.clear();
      for (int i = 0; i < V * 4; ++i) h.push_back(__float2half(small(9000 + i) / 8.0f));
      if (slot == 1) h[77] = __float2half(NAN);
      b.fill(h);
      head.SetAdapter(slot, a.p, IN, b.p, 4, 4, 0.5f, st);
      cudaStreamSynchronize(st);
    }
  }
  ~Bench() { cudaStreamDestroy(st); }
  std::vector<GenerationResult> run(const std::vector<BatchRequest>& rq, const std::vector<Random*>& randoms = {}) {
    return gen.GenerateBatch(
        [this](const std::vector<std::vector<int>>& contexts, cudaStream_t stream) {
          std::vector<__half> rows;
          for (const auto& c : contexts) {
            uint64_t z = 0;
            for (int t : c) z = z * 31 + t + 1;
            const bool bad = c[0] == poisoned && c.size() >= from;
            for (int i = 0; i < IN; ++i) rows.push_back(__float2half(bad ? NAN : static_cast<float>(small(z + i))));
          }
          cudaMemcpyAsync(x.p, rows.data(), rows.size() * 2, cudaMemcpyHostToDevice, stream);
          cudaStreamSynchronize(stream);
          return static_cast<const void*>(x.p);
        },
        head, rq, st, randoms);
  }
};

static const std::vector<int> none;
static GenerationOptions sampled(int seed, float T = 0.9f) {
  return GenerationOptions::Create(false, T, 0.95f, 40, 1.0f, 12, none, seed);
}

static void largest_draw(Bench& t) {
  Fixed top(1.0 - 0x1p-26), low(0.25);
  const auto r = t.run({{{3, 1}, sampled(1), 0.0f, 0}, {{4}, sampled(2), 0.0f, -1}}, {&top, &low});
  EXPECT(r[0].GeneratedTokenIds.size() == 12 && r[1].GeneratedTokenIds.size() == 12, "a draw next to 1 gives a token");
  for (int token : r[0].GeneratedTokenIds) EXPECT(token >= 0 && token < V, "a token of the vocabulary");
}

static bool same(const GenerationResult& a, const GenerationResult& b) {
  return a.GeneratedTokenIds == b.GeneratedTokenIds && a.FinishReason == b.FinishReason && a.Flags == b.Flags;
}

static void one_of_many(Bench& t) {
  const std::vector<BatchRequest> sound = {{{3, 1}, sampled(1), 0.0f, 0},
                                           {{4}, GenerationOptions::CreateGreedy(9, none), 0.0f, -1},
                                           {{5, 5}, sampled(3), 0.1f, 0}};
  const auto want = t.run(sound);
  for (const auto& r : want) EXPECT(r.FinishReason == GenerationFinishReason::MaxNewTokens && r.Flags == 0, "sound requests");
  // an adapter with a NaN, a hidden state that becomes NaN, and options out of range, among them
  t.poisoned = 250;
  t.from = 4;
  std::vector<BatchRequest> rq = {sound[0], {{8, 2}, sampled(4), 0.0f, 1}, sound[1], {{250}, sampled(5), 0.0f, 0}, sound[2],
                                  {{6}, sampled(6, NAN), 0.0f, -1}, {{7}, GenerationOptions::CreateGreedy(3, none), 0.0f, 1}};
  const auto r = t.run(rq);
  EXPECT(same(r[0], want[0]) && same(r[2], want[1]) && same(r[4], want[2]), "the others' tokens are as without them");
  for (size_t i : {size_t{1}, size_t{6}})
    EXPECT(r[i].FinishReason == GenerationFinishReason::Failed && r[i].Flags == NCB_FLAG_NONFINITE &&
               r[i].GeneratedTokenIds.empty(), "an adapter with a NaN fails its request");
  EXPECT(r[3].FinishReason == GenerationFinishReason::Failed && r[3].Flags == NCB_FLAG_NONFINITE &&
             r[3].GeneratedTokenIds.size() == 3, "a request that fails later keeps its tokens");
  EXPECT(r[5].FinishReason == GenerationFinishReason::Failed && r[5].Flags == NCB_FLAG_BAD_OPTIONS, "options out of range");
  t.poisoned = -1;
  const auto alone = t.run({rq[1]});
  EXPECT(alone.size() == 1 && alone[0].FinishReason == GenerationFinishReason::Failed, "the last request running fails");
}

static void a_kernel_gave_up(Bench& t) {
  g_status = NCB_ERROR_LAUNCH_FAILED;
  int status = NCB_OK;
  try {
    t.run({{{3, 1}, sampled(1), 0.0f, 0}});
  } catch (const CudaException& e) {
    status = e.status;
  }
  EXPECT(status == NCB_ERROR_LAUNCH_FAILED, "undefined logits are not sampled on");
  g_status = NCB_OK;
  EXPECT(t.run({{{3, 1}, sampled(1), 0.0f, 0}})[0].GeneratedTokenIds.size() == 12, "and as before without");
}

static void a_refused_call(Bench& t) {
  g_refuse = true;
  int status = NCB_OK;
  try {
    t.run({{{3, 1}, sampled(1), 0.0f, 0}});
  } catch (const CudaException& e) {
    status = e.status;
  }
  g_refuse = false;
  EXPECT(status == NCB_ERROR_CAPACITY && g_ended && cudaStreamQuery(t.st) == cudaSuccess, "nothing is left on the stream");
}

int main(int argc, char** argv) {
  draw_tests();
  if (argc < 2 || std::strcmp(argv[1], "--no-gpu") != 0) {
    Bench t;
    largest_draw(t);
    one_of_many(t);
    a_kernel_gave_up(t);
    a_refused_call(t);
  }
  std::printf("%d checks, %d failed\n", g_run, g_fail);
  return g_fail == 0 ? 0 : 1;
}
