// C++ mirror of the reference's generation interface for the sampling path
// (Neuraval.Core.Generation: GenerationOptions, TokenSampler, LogitsProcessor;
// Neuraval/Generation/*.cs) over libnavsampler's C ABI (navsampler.h). Same
// names, argument meaning and argument checks, in the same order, with the
// exception types of the C# code:
//   ArgumentException           -> neuraval::ArgumentException
//   ArgumentNullException       -> neuraval::ArgumentNullException
//   ArgumentOutOfRangeException -> neuraval::ArgumentOutOfRangeException
//   CudaException               -> neuraval::CudaException (a non-OK status)
// C# references become pointers where the reference checks them for null
// (the pointer overloads), with reference overloads for ordinary use.
// The C# classes are static; here a Device owns the sampler handle (device
// scratch), and TokenSampler / LogitsProcessor borrow it.
#pragma once

#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstring>
#include <functional>
#include <memory>
#include <optional>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "navsampler.h"

namespace neuraval {

struct ArgumentException : std::invalid_argument {
  explicit ArgumentException(const std::string& param) : std::invalid_argument(param) {}
};
struct ArgumentNullException : std::invalid_argument {
  explicit ArgumentNullException(const std::string& param) : std::invalid_argument(param) {}
};
struct ArgumentOutOfRangeException : std::out_of_range {
  explicit ArgumentOutOfRangeException(const std::string& param) : std::out_of_range(param) {}
};
struct CudaException : std::runtime_error {
  int status;
  CudaException(int st, const std::string& where)
      : std::runtime_error(where + ": " + ncb_sampler_status_message(st)), status(st) {}
};

inline void check(int st, const char* where) {
  if (st != NCB_OK) throw CudaException(st, where);
}

// GenerationOptions (GenerationOptions.cs:5-98) plus the new frequency and
// presence penalties (0 = off).
class GenerationOptions {
 public:
  bool Greedy() const { return greedy_; }
  float Temperature() const { return temperature_; }
  float TopP() const { return top_p_; }
  int TopK() const { return top_k_; }
  float RepetitionPenalty() const { return repetition_penalty_; }
  int MaxNewTokens() const { return max_new_tokens_; }
  const std::vector<int>& StopTokenIds() const { return stop_token_ids_; }
  std::optional<int> Seed() const { return seed_; }
  float FrequencyPenalty() const { return frequency_penalty_; }
  float PresencePenalty() const { return presence_penalty_; }

  // GenerationOptions.Create (:44-75): the same checks in the same order.
  static GenerationOptions Create(bool greedy, float temperature, float topP, int topK,
                                  float repetitionPenalty, int maxNewTokens,
                                  const std::vector<int>* stopTokenIds,
                                  std::optional<int> seed = std::nullopt) {
    if (temperature <= 0.0f) throw ArgumentOutOfRangeException("temperature");
    if (topP <= 0.0f || topP > 1.0f) throw ArgumentOutOfRangeException("topP");
    if (topK <= 0) throw ArgumentOutOfRangeException("topK");
    if (repetitionPenalty <= 0.0f) throw ArgumentOutOfRangeException("repetitionPenalty");
    if (maxNewTokens <= 0) throw ArgumentOutOfRangeException("maxNewTokens");
    if (!stopTokenIds) throw ArgumentNullException("stopTokenIds");
    GenerationOptions o;
    o.greedy_ = greedy;
    o.temperature_ = temperature;
    o.top_p_ = topP;
    o.top_k_ = topK;
    o.repetition_penalty_ = repetitionPenalty;
    o.max_new_tokens_ = maxNewTokens;
    o.stop_token_ids_ = *stopTokenIds;
    o.seed_ = seed;
    return o;
  }
  static GenerationOptions Create(bool greedy, float temperature, float topP, int topK,
                                  float repetitionPenalty, int maxNewTokens,
                                  const std::vector<int>& stopTokenIds,
                                  std::optional<int> seed = std::nullopt) {
    return Create(greedy, temperature, topP, topK, repetitionPenalty, maxNewTokens,
                  &stopTokenIds, seed);
  }
  // GenerationOptions.CreateGreedy (:77-80) and Default (:82-85).
  static GenerationOptions CreateGreedy(int maxNewTokens, const std::vector<int>& stopTokenIds,
                                        std::optional<int> seed = std::nullopt) {
    return Create(true, 1.0f, 1.0f, INT_MAX, 1.0f, maxNewTokens, stopTokenIds, seed);
  }
  static GenerationOptions Default(const std::vector<int>& stopTokenIds,
                                   std::optional<int> seed = std::nullopt) {
    return Create(false, 0.7f, 0.9f, 40, 1.1f, 256, stopTokenIds, seed);
  }
  // New: a copy with frequency and presence penalties (applied after the
  // repetition penalty, before the temperature).
  GenerationOptions WithPenalties(float frequency, float presence) const {
    GenerationOptions o = *this;
    o.frequency_penalty_ = frequency;
    o.presence_penalty_ = presence;
    return o;
  }

  NcbSamplerParams ToParams() const {
    NcbSamplerParams p{};
    p.greedy = greedy_ ? 1 : 0;
    p.temperature = temperature_;
    p.top_p = top_p_;
    p.top_k = top_k_;
    p.repetition_penalty = repetition_penalty_;
    p.frequency_penalty = frequency_penalty_;
    p.presence_penalty = presence_penalty_;
    return p;
  }

 private:
  GenerationOptions() = default;
  bool greedy_ = false;
  float temperature_ = 1.0f, top_p_ = 1.0f;
  int top_k_ = INT_MAX;
  float repetition_penalty_ = 1.0f;
  int max_new_tokens_ = 1;
  std::vector<int> stop_token_ids_;
  std::optional<int> seed_;
  float frequency_penalty_ = 0.0f, presence_penalty_ = 0.0f;
};

// The uniform source of the draw: TokenSampler.cs:125 uses
// (float)random.NextDouble(). Any generator with NextDouble() in [0, 1) fits.
struct Random {
  virtual ~Random() = default;
  virtual double NextDouble() = 0;
};
class DefaultRandom final : public Random {
 public:
  explicit DefaultRandom(uint64_t seed = 0) : gen_(seed) {}
  double NextDouble() override { return std::uniform_real_distribution<double>(0.0, 1.0)(gen_); }

 private:
  std::mt19937_64 gen_;
};

// A draw as ncb_sample_rows_min_p_device takes it, in [0, 1): doubles from 1 - 2^-25 on
// would round to 1.
inline float UniformBelowOne(double u) { return std::min(static_cast<float>(u), 1.0f - 0x1p-24f); }

// One GPU's sampler handle (ncb_sampler_create): scratch for up to maxRows rows
// of up to maxVocab columns and maxHistory generated ids per row.
class Device {
 public:
  explicit Device(int device = 0, int maxRows = 1, int maxVocab = 262144, int maxHistory = 4096) {
    check(ncb_sampler_create(device, maxRows, maxVocab, maxHistory, &h_), "ncb_sampler_create");
  }
  ~Device() {
    if (h_) ncb_sampler_destroy(h_);
  }
  Device(const Device&) = delete;
  Device& operator=(const Device&) = delete;
  NcbSampler* handle() const { return h_; }

 private:
  NcbSampler* h_ = nullptr;
};

// TokenSampler (TokenSampler.cs:10-143) on the GPU.
class TokenSampler {
 public:
  explicit TokenSampler(Device& device) : d_(device) {}

  // TokenSampler.SampleNext (:10-30): argument checks in the reference's order,
  // then one row through ncb_sample_rows. A non-finite row (NaN/+inf, no finite
  // maximum) or a history beyond the handle's capacity throws CudaException.
  int SampleNext(const std::vector<float>* logits, const GenerationOptions* options,
                 const std::vector<int>* generatedTokenIds, Random* random) const {
    if (!logits) throw ArgumentNullException("logits");
    if (!options) throw ArgumentNullException("options");
    if (!generatedTokenIds) throw ArgumentNullException("generatedTokenIds");
    if (!random) throw ArgumentNullException("random");
    const NcbSamplerParams p = options->ToParams();
    // the reference draws only on the filtered path (:125)
    const float u = options->Greedy() ? 0.0f : static_cast<float>(random->NextDouble());
    const int32_t offsets[2] = {0, static_cast<int32_t>(generatedTokenIds->size())};
    int32_t token = -1;
    uint32_t flags = 0;
    check(ncb_sample_rows(d_.handle(), logits->data(), 1, static_cast<int>(logits->size()),
                          generatedTokenIds->empty() ? nullptr : generatedTokenIds->data(),
                          offsets, &u, &p, &token, &flags, nullptr),
          "ncb_sample_rows");
    if (token < 0) throw CudaException(NCB_ERROR_INVALID_ARGUMENT, "SampleNext: row not sampled");
    return token;
  }
  int SampleNext(const std::vector<float>& logits, const GenerationOptions& options,
                 const std::vector<int>& generatedTokenIds, Random& random) const {
    return SampleNext(&logits, &options, &generatedTokenIds, &random);
  }

  // Batched form: rows x vocab logits (row-major), one history per row. Each
  // row consumes one NextDouble() unless greedy, in row order.
  std::vector<int> SampleNextBatch(const std::vector<float>& logits, int rows,
                                   const GenerationOptions& options,
                                   const std::vector<std::vector<int>>& generatedTokenIds,
                                   Random& random, std::vector<uint32_t>* flagsOut = nullptr) const {
    if (rows < 0 || (rows > 0 && logits.size() % rows != 0) ||
        generatedTokenIds.size() != static_cast<size_t>(rows))
      throw ArgumentOutOfRangeException("rows");
    std::vector<int32_t> offsets(rows + 1, 0), hist;
    for (int r = 0; r < rows; ++r) {
      hist.insert(hist.end(), generatedTokenIds[r].begin(), generatedTokenIds[r].end());
      offsets[r + 1] = static_cast<int32_t>(hist.size());
    }
    std::vector<float> u(rows, 0.0f);
    if (!options.Greedy())
      for (float& x : u) x = static_cast<float>(random.NextDouble());
    std::vector<int32_t> tokens(rows, -1);
    std::vector<uint32_t> flags(rows, 0);
    const NcbSamplerParams p = options.ToParams();
    const int vocab = rows > 0 ? static_cast<int>(logits.size() / rows) : 1;
    check(ncb_sample_rows(d_.handle(), logits.data(), rows, vocab, hist.empty() ? nullptr : hist.data(),
                          offsets.data(), u.data(), &p, tokens.data(), flags.data(), nullptr),
          "ncb_sample_rows");
    if (flagsOut) *flagsOut = flags;
    return std::vector<int>(tokens.begin(), tokens.end());
  }

 private:
  Device& d_;
};

// LogitsProcessor (LogitsProcessor.cs:8-114) on the GPU, in place.
class LogitsProcessor {
 public:
  explicit LogitsProcessor(Device& device) : d_(device) {}

  // ApplyRepetitionPenalty (:8-36)
  void ApplyRepetitionPenalty(std::vector<float>* logits, const std::vector<int>* generatedTokenIds,
                              float penalty) const {
    if (!logits) throw ArgumentNullException("logits");
    if (!generatedTokenIds) throw ArgumentNullException("generatedTokenIds");
    if (penalty <= 0.0f) throw ArgumentOutOfRangeException("penalty");
    if (penalty == 1.0f || generatedTokenIds->empty() || logits->empty()) return;
    const int32_t offsets[2] = {0, static_cast<int32_t>(generatedTokenIds->size())};
    check(ncb_logits_repetition_penalty(d_.handle(), logits->data(), 1,
                                        static_cast<int>(logits->size()), generatedTokenIds->data(),
                                        offsets, penalty),
          "ncb_logits_repetition_penalty");
  }
  // ApplyTemperature (:38-51)
  void ApplyTemperature(std::vector<float>* logits, float temperature) const {
    if (!logits) throw ArgumentNullException("logits");
    if (temperature <= 0.0f) throw ArgumentOutOfRangeException("temperature");
    if (temperature == 1.0f || logits->empty()) return;
    check(ncb_logits_temperature(d_.handle(), logits->data(), 1, static_cast<int>(logits->size()),
                                 temperature),
          "ncb_logits_temperature");
  }
  // FilterTopK (:53-73)
  void FilterTopK(std::vector<float>* logits, int topK) const {
    if (!logits) throw ArgumentNullException("logits");
    if (topK <= 0) throw ArgumentOutOfRangeException("topK");
    if (topK >= static_cast<int>(logits->size())) return;
    check(ncb_logits_filter_top_k(d_.handle(), logits->data(), 1, static_cast<int>(logits->size()),
                                  topK),
          "ncb_logits_filter_top_k");
  }
  // FilterTopP (:75-114)
  void FilterTopP(std::vector<float>* probabilities, float topP) const {
    if (!probabilities) throw ArgumentNullException("probabilities");
    if (topP <= 0.0f || topP > 1.0f) throw ArgumentOutOfRangeException("topP");
    if (topP >= 1.0f || probabilities->empty()) return;
    check(ncb_logits_filter_top_p(d_.handle(), probabilities->data(), 1,
                                  static_cast<int>(probabilities->size()), topP, nullptr),
          "ncb_logits_filter_top_p");
  }

 private:
  Device& d_;
};

// The LM head with each request's low-rank adapter (ncb_adapter_head_*): what
// ModernDecoderModel.ComputeLogits (ModernDecoderModel.cs:221-240) does for one
// request, for the rows of many. dtype: NCB_DTYPE_F16 or NCB_DTYPE_BF16; all
// pointers are device pointers, everything is ordered on the given stream.
class AdapterHead {
 public:
  AdapterHead(int device, int dtype, int inFeatures, int outFeatures, int maxRows, int maxAdapters = 0,
              int maxRank = 0)
      : device_(device), in_(inFeatures), out_(outFeatures), max_rows_(maxRows) {
    check(ncb_adapter_head_create(device, dtype, inFeatures, outFeatures, maxRows, maxAdapters,
                                  maxRank, &h_),
          "ncb_adapter_head_create");
  }
  ~AdapterHead() {
    if (h_) ncb_adapter_head_destroy(h_);
  }
  AdapterHead(const AdapterHead&) = delete;
  AdapterHead& operator=(const AdapterHead&) = delete;
  int DeviceId() const { return device_; }
  int InFeatures() const { return in_; }
  int OutFeatures() const { return out_; }
  int MaxRows() const { return max_rows_; }

  // [outFeatures, inFeatures], rows ld apart; stays the caller's and in use.
  void SetWeight(const void* weight, int64_t ld, cudaStream_t stream) const {
    check(ncb_adapter_head_set_weight_device(h_, weight, ld, stream),
          "ncb_adapter_head_set_weight_device");
  }
  // a [rank, inFeatures] and b [outFeatures, rank] are copied.
  void SetAdapter(int slot, const void* a, int64_t lda, const void* b, int64_t ldb, int rank,
                  float scale, cudaStream_t stream) const {
    check(ncb_adapter_head_set_adapter_device(h_, slot, a, lda, b, ldb, rank, scale, stream),
          "ncb_adapter_head_set_adapter_device");
  }
  void ClearAdapter(int slot, cudaStream_t stream) const {
    check(ncb_adapter_head_clear_adapter_device(h_, slot, stream),
          "ncb_adapter_head_clear_adapter_device");
  }
  // CudaException if a wait inside one of the head's kernels gave up; to be called once
  // the stream has been synchronised.
  void Check() const { check(ncb_adapter_head_status(h_), "ncb_adapter_head_status"); }
  // out [rows, outFeatures] of outDtype from x [rows, inFeatures]; adapterIds: a slot
  // per row (-1: none), or nullptr.
  void Project(const void* x, int64_t ldx, int rows, const int32_t* adapterIds, void* out,
               int outDtype, int64_t ldo, cudaStream_t stream) const {
    check(ncb_adapter_head_project_device(h_, x, ldx, rows, adapterIds, out, outDtype, ldo, stream),
          "ncb_adapter_head_project_device");
  }

 private:
  NcbAdapterHead* h_ = nullptr;
  int device_, in_, out_, max_rows_;
};

// One request of TextGenerator::GenerateBatch: the reference's prompt and options,
// and two settings it does not have, a min-p and the adapter slot of the head.
struct BatchRequest {
  std::vector<int> PromptTokenIds;
  GenerationOptions Options;
  float MinP = 0.0f;
  int Adapter = -1;
};

// GenerationFinishReason (GenerationFinishReason.cs) and GenerationResult
// (GenerationResult.cs:7-27). Failed and Flags are GenerateBatch's, for a request that
// ended without a token to go on with: NCB_FLAG_NONFINITE or NCB_FLAG_BAD_OPTIONS. The
// tokens before that are there.
enum class GenerationFinishReason { MaxNewTokens, StopToken, Failed };
struct GenerationResult {
  std::vector<int> GeneratedTokenIds;
  GenerationFinishReason FinishReason = GenerationFinishReason::MaxNewTokens;
  uint32_t Flags = 0;
};

// TextGenerator.Generate (TextGenerator.cs:19-51): the decode loop around
// TokenSampler.SampleNext. The model is a callable from the context window's
// token ids to the last position's logits (_model.Forward followed by
// ExtractLastPositionLogits, :34-35); the context is the sequence trimmed to
// the model's last maxPositionEmbeddings ids (TrimToContextWindow,
// :128-139). The history passed to the sampler is the generated ids only
// (:37), and the random source is drawn once per non-greedy step and never
// on a greedy step (TokenSampler.cs:125). Without a random source the loop
// seeds its own from options.Seed(), as :26 does (a std::mt19937_64, not
// .NET's Random: the draws differ from the reference's for the same seed).
class TextGenerator {
 public:
  using Model = std::function<std::vector<float>(const std::vector<int>& context)>;
  // The device-resident handoff: the model leaves the last position's logits
  // in device memory it owns (`vocab` floats, complete in stream order on
  // `stream`) and returns their address; the sampler reads them in place
  // (the D2H copy of ModernDecoderModel.cs:169-170 is gone).
  using DeviceModel = std::function<const float*(const std::vector<int>& context,
                                                 cudaStream_t stream)>;

  TextGenerator(Device& device, int maxPositionEmbeddings)
      : device_(device), sampler_(device), max_positions_(maxPositionEmbeddings) {
    if (maxPositionEmbeddings < 1) throw ArgumentOutOfRangeException("maxPositionEmbeddings");
  }

  GenerationResult Generate(const Model& model, const std::vector<int>& promptTokenIds,
                            const GenerationOptions& options, Random* random = nullptr) const {
    if (!model) throw ArgumentNullException("model");
    if (promptTokenIds.empty()) throw ArgumentException("promptTokenIds");
    std::optional<DefaultRandom> own;
    if (!random) random = &own.emplace(SeedOf(options));
    std::vector<int> sequence(promptTokenIds), generated;
    GenerationResult result;
    for (int step = 0; step < options.MaxNewTokens(); ++step) {
      const std::vector<float> logits = model(Trim(sequence));
      const int next = sampler_.SampleNext(logits, options, generated, *random);
      generated.push_back(next);
      sequence.push_back(next);
      if (IsStop(options, next)) {
        result.FinishReason = GenerationFinishReason::StopToken;
        break;
      }
    }
    result.GeneratedTokenIds = std::move(generated);
    return result;
  }

  // Generate with the logits left on the device. Per step: the model's
  // launches, one 12-byte copy to the device (the history length and the
  // uniform, from pinned memory), ncb_sample_rows_device writing the token
  // straight into the device history (its next slot), and one 4-byte copy
  // back for the stop test and the next context.
  GenerationResult GenerateDevice(const DeviceModel& model, int vocab,
                                  const std::vector<int>& promptTokenIds,
                                  const GenerationOptions& options, cudaStream_t stream,
                                  Random* random = nullptr) const {
    if (!model) throw ArgumentNullException("model");
    if (promptTokenIds.empty()) throw ArgumentException("promptTokenIds");
    if (vocab <= 0) throw ArgumentOutOfRangeException("vocab");
    std::optional<DefaultRandom> own;
    if (!random) random = &own.emplace(SeedOf(options));
    const int cap = std::max(1, options.MaxNewTokens());
    auto dev_free = [](void* p) { cudaFree(p); };
    auto host_free = [](void* p) { cudaFreeHost(p); };
    void* p = nullptr;
    cuda(cudaMalloc(&p, sizeof(int32_t) * (size_t)(cap + 4)), "cudaMalloc");
    std::unique_ptr<void, decltype(dev_free)> dmem(p, dev_free);
    p = nullptr;
    cuda(cudaMallocHost(&p, sizeof(int32_t) * 4), "cudaMallocHost");
    std::unique_ptr<void, decltype(host_free)> hmem(p, host_free);
    int32_t* d_hist = static_cast<int32_t*>(dmem.get());  // [cap] generated ids
    int32_t* d_step = d_hist + cap;                       // {0, n, bits of u}
    int32_t* h_step = static_cast<int32_t*>(hmem.get());  // pinned {0, n, u, token}
    const NcbSamplerParams prm = options.ToParams();
    std::vector<int> sequence(promptTokenIds), generated;
    GenerationResult result;
    for (int step = 0; step < options.MaxNewTokens(); ++step) {
      const float* d_logits = model(Trim(sequence), stream);
      if (!d_logits) throw ArgumentNullException("logits");
      const float u = options.Greedy() ? 0.0f : static_cast<float>(random->NextDouble());
      h_step[0] = 0;
      h_step[1] = step;
      std::memcpy(&h_step[2], &u, sizeof(float));
      cuda(cudaMemcpyAsync(d_step, h_step, 3 * sizeof(int32_t), cudaMemcpyHostToDevice, stream),
           "cudaMemcpyAsync");
      check(ncb_sample_rows_device(device_.handle(), d_logits, 1, vocab, d_hist, d_step,
                                   reinterpret_cast<const float*>(d_step + 2), &prm,
                                   d_hist + step, nullptr, nullptr, stream),
            "ncb_sample_rows_device");
      cuda(cudaMemcpyAsync(&h_step[3], d_hist + step, sizeof(int32_t), cudaMemcpyDeviceToHost,
                           stream),
           "cudaMemcpyAsync");
      cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
      const int next = h_step[3];
      if (next < 0) throw CudaException(NCB_ERROR_INVALID_ARGUMENT, "GenerateDevice: row not sampled");
      generated.push_back(next);
      sequence.push_back(next);
      if (IsStop(options, next)) {
        result.FinishReason = GenerationFinishReason::StopToken;
        break;
      }
    }
    result.GeneratedTokenIds = std::move(generated);
    return result;
  }

  // The last hidden states of the given contexts, [contexts, in_features] of the
  // head's type in device memory, complete in stream order on `stream`.
  using HiddenModel = std::function<const void*(const std::vector<std::vector<int>>& contexts,
                                                cudaStream_t stream)>;

  // Generate for many requests in step, each with options, random source and
  // adapter of its own: per step the model's hidden states of the requests still
  // running, the head's projection with their adapters and one sampling call with
  // their options; 24 bytes per request go to the device and 8 come back.
  // `randoms`: a source per request, or empty (each request then seeds its own).
  // A request's tokens do not depend on the others': one whose logits are not finite
  // (its hidden state, its adapter, a product past fp16's range) or whose options the
  // sampling call does not take ends as Failed, alone. ncb_sample_rows_min_p_device
  // knows no history of tokens, so a request that sets a repetition, frequency or
  // presence penalty (GenerationOptions::Default does) is refused; Generate takes it.
  std::vector<GenerationResult> GenerateBatch(const HiddenModel& model, const AdapterHead& head,
                                              const std::vector<BatchRequest>& requests,
                                              cudaStream_t stream,
                                              const std::vector<Random*>& randoms = {}) const {
    if (!model) throw ArgumentNullException("model");
    if (requests.empty()) return {};
    if (static_cast<int>(requests.size()) > head.MaxRows()) throw ArgumentOutOfRangeException("requests");
    if (!randoms.empty() && randoms.size() != requests.size()) throw ArgumentException("randoms");
    for (const BatchRequest& r : requests) {
      if (r.PromptTokenIds.empty()) throw ArgumentException("promptTokenIds");
      if (!(r.MinP >= 0.0f && r.MinP <= 1.0f)) throw ArgumentOutOfRangeException("minP");
      if (r.Options.RepetitionPenalty() != 1.0f || r.Options.FrequencyPenalty() != 0.0f ||
          r.Options.PresencePenalty() != 0.0f)
        throw ArgumentException("options");
    }
    const size_t n = requests.size(), vocab = static_cast<size_t>(head.OutFeatures());
    int before = 0;
    cuda(cudaGetDevice(&before), "cudaGetDevice");
    cuda(cudaSetDevice(head.DeviceId()), "cudaSetDevice");
    const auto restore = [before](void*) { cudaSetDevice(before); };
    std::unique_ptr<void, decltype(restore)> device(this_address(), restore);
    auto dev_free = [](void* p) { cudaFree(p); };
    auto host_free = [](void* p) { cudaFreeHost(p); };
    // per request: adapter, T, top_k, top_p, min_p, u; then the token and its flags
    void* p = nullptr;
    cuda(cudaMalloc(&p, 8 * 4 * n), "cudaMalloc");
    std::unique_ptr<void, decltype(dev_free)> dmem(p, dev_free);
    p = nullptr;
    cuda(cudaMalloc(&p, sizeof(float) * n * vocab), "cudaMalloc");
    std::unique_ptr<void, decltype(dev_free)> logits(p, dev_free);
    p = nullptr;
    cuda(cudaMallocHost(&p, 8 * 4 * n), "cudaMallocHost");
    std::unique_ptr<void, decltype(host_free)> hmem(p, host_free);
    // an exception may leave copies on the stream: they end before their buffers do
    const auto wait = [stream](void*) { cudaStreamSynchronize(stream); };
    std::unique_ptr<void, decltype(wait)> idle(this_address(), wait);
    int32_t* d = static_cast<int32_t*>(dmem.get());
    int32_t* h = static_cast<int32_t*>(hmem.get());
    std::vector<std::optional<DefaultRandom>> own(n);
    std::vector<Random*> random(n);
    for (size_t i = 0; i < n; ++i)
      random[i] = randoms.empty() || !randoms[i] ? &own[i].emplace(SeedOf(requests[i].Options)) : randoms[i];
    std::vector<std::vector<int>> sequences(n);
    std::vector<GenerationResult> results(n);
    std::vector<size_t> running;
    for (size_t i = 0; i < n; ++i) {
      sequences[i] = requests[i].PromptTokenIds;
      if (requests[i].Options.MaxNewTokens() > 0) running.push_back(i);
    }
    while (!running.empty()) {
      const size_t rows = running.size();
      std::vector<std::vector<int>> contexts;
      for (size_t i : running) contexts.push_back(Trim(sequences[i]));
      const void* hidden = model(contexts, stream);
      if (!hidden) throw ArgumentNullException("hidden");
      for (size_t j = 0; j < rows; ++j) {
        const BatchRequest& r = requests[running[j]];
        const bool greedy = r.Options.Greedy();
        const float T = greedy ? 0.0f : r.Options.Temperature(), top_p = r.Options.TopP(),
                    u = greedy ? 0.0f : UniformBelowOne(random[running[j]]->NextDouble());
        h[j] = r.Adapter;
        std::memcpy(h + rows + j, &T, 4);
        h[2 * rows + j] = r.Options.TopK();
        std::memcpy(h + 3 * rows + j, &top_p, 4);
        std::memcpy(h + 4 * rows + j, &r.MinP, 4);
        std::memcpy(h + 5 * rows + j, &u, 4);
      }
      cuda(cudaMemcpyAsync(d, h, 6 * 4 * rows, cudaMemcpyHostToDevice, stream), "cudaMemcpyAsync");
      head.Project(hidden, head.InFeatures(), static_cast<int>(rows), d, logits.get(), NCB_DTYPE_F32,
                   static_cast<int64_t>(vocab), stream);
      const float* f = reinterpret_cast<const float*>(d);
      check(ncb_sample_rows_min_p_device(logits.get(), NCB_DTYPE_F32, static_cast<int>(rows),
                                         static_cast<int>(vocab), static_cast<int64_t>(vocab),
                                         f + 5 * rows, f + rows, d + 2 * rows, f + 3 * rows,
                                         f + 4 * rows, d + 6 * rows, nullptr, nullptr,
                                         reinterpret_cast<uint32_t*>(d + 7 * rows), stream),
            "ncb_sample_rows_min_p_device");
      cuda(cudaMemcpyAsync(h + 6 * rows, d + 6 * rows, 2 * 4 * rows, cudaMemcpyDeviceToHost, stream),
           "cudaMemcpyAsync");
      cuda(cudaStreamSynchronize(stream), "cudaStreamSynchronize");
      head.Check();
      std::vector<size_t> still;
      for (size_t j = 0; j < rows; ++j) {
        const size_t i = running[j];
        const int next = h[6 * rows + j];
        if (next < 0) {
          results[i].FinishReason = GenerationFinishReason::Failed;
          results[i].Flags = static_cast<uint32_t>(h[7 * rows + j]);
          continue;
        }
        results[i].GeneratedTokenIds.push_back(next);
        sequences[i].push_back(next);
        if (IsStop(requests[i].Options, next))
          results[i].FinishReason = GenerationFinishReason::StopToken;
        else if (static_cast<int>(results[i].GeneratedTokenIds.size()) < requests[i].Options.MaxNewTokens())
          still.push_back(i);
      }
      running.swap(still);
    }
    return results;
  }

 private:
  static void* this_address() {  // anything but null: a unique_ptr calls its deleter for it
    static char c;
    return &c;
  }
  static uint64_t SeedOf(const GenerationOptions& o) {
    return o.Seed() ? static_cast<uint64_t>(*o.Seed()) : std::random_device{}();
  }
  static bool IsStop(const GenerationOptions& o, int token) {
    const std::vector<int>& s = o.StopTokenIds();
    return std::find(s.begin(), s.end(), token) != s.end();
  }
  static void cuda(cudaError_t e, const char* where) {
    if (e != cudaSuccess) throw CudaException(NCB_ERROR_LAUNCH_FAILED, where);
  }
  std::vector<int> Trim(const std::vector<int>& sequence) const {
    if ((int)sequence.size() <= max_positions_) return sequence;
    return std::vector<int>(sequence.end() - max_positions_, sequence.end());
  }

  Device& device_;
  TokenSampler sampler_;
  int max_positions_;
};

}  // namespace neuraval
