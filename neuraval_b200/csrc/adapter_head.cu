// LM head with low-rank adapters of many requests (sm_100a):
//   out[n, :] = W x_n + scale_s B_s (A_s x_n),  s = adapter_ids[n].
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <mutex>
#include <new>

#include "navsampler.h"

int ncb_record_status(int st);

namespace nvs {

constexpr int AH_MAX_ADAPTERS = 1024;
constexpr int AH_MAX_RANK = 128;

struct AhArgs {
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  int rows, in, out, slots, rpad;
  const int32_t* ids;
  const void* a;        // [slots][rpad][in]
  const void* b;        // [slots][out][rpad]
  const int32_t* ranks; // per slot, 0: empty
  const float* scales;
  float* u;             // [rows][rpad]
  void* y;
  int64_t ldo;
};

template <typename E>
__device__ __forceinline__ float ah_float(E v) { return (float)v; }

template <typename E>
__global__ void adapter_pack_kernel(E* a, E* b, int32_t* ranks, float* scales, int slot, int in,
                                    int out, int rpad, const E* sa, int64_t lda, const E* sb,
                                    int64_t ldb, int rank, float scale) {
  const int64_t na = (int64_t)rpad * in, nb = (int64_t)out * rpad;
  const int64_t t0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x, dt = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = t0; i < na; i += dt) {
    const int64_t j = i / in, k = i % in;
    a[slot * na + i] = j < rank ? sa[j * lda + k] : E(0.0f);
  }
  for (int64_t i = t0; i < nb; i += dt) {
    const int64_t v = i / rpad, j = i % rpad;
    b[slot * nb + i] = j < rank ? sb[v * ldb + j] : E(0.0f);
  }
  if (t0 == 0) {
    ranks[slot] = rank;
    scales[slot] = scale;
  }
}

// u[n][j] = scale A_s[j] x_n, a warp for each.
template <typename E>
__global__ void adapter_shrink_kernel(const AhArgs g) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  if (at >= (int64_t)g.rows * g.rpad) return;
  const int n = (int)(at / g.rpad), j = (int)(at % g.rpad), s = g.ids[n];
  float sum = 0.0f;
  if (s >= 0 && s < g.slots && j < g.ranks[s]) {
    const E* x = static_cast<const E*>(g.x) + n * g.ldx;
    const E* a = static_cast<const E*>(g.a) + ((int64_t)s * g.rpad + j) * g.in;
    for (int k = lane; k < g.in; k += 32) sum = fmaf(ah_float(x[k]), ah_float(a[k]), sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum *= g.scales[s];
  }
  if (lane == 0) g.u[at] = sum;
}

// 64 rows by 64 columns of the output per block, 4 x 4 per thread.
template <typename E, typename O>
__global__ void __launch_bounds__(256) adapter_project_kernel(const AhArgs g) {
  __shared__ float sx[16][65], sw[16][65];
  const int n0 = blockIdx.y * 64, v0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.in; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, k = k0 + (i & 15);
      sx[i & 15][r] = n0 + r < g.rows && k < g.in
                          ? ah_float(static_cast<const E*>(g.x)[(n0 + r) * g.ldx + k]) : 0.0f;
      sw[i & 15][r] = v0 + r < g.out && k < g.in
                          ? ah_float(static_cast<const E*>(g.w)[(v0 + r) * g.ldw + k]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(sx[k][ty + 16 * i], sw[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + ty + 16 * i;
    if (n >= g.rows) continue;
    const int s = g.ids ? g.ids[n] : -1;
    const int rank = s >= 0 && s < g.slots ? g.ranks[s] : 0;
    for (int j = 0; j < 4; ++j) {
      const int v = v0 + tx + 16 * j;
      if (v >= g.out) continue;
      float y = acc[i][j];
      const E* b = static_cast<const E*>(g.b) + ((int64_t)s * g.out + v) * g.rpad;
      for (int r = 0; r < rank; ++r) y = fmaf(ah_float(b[r]), g.u[(int64_t)n * g.rpad + r], y);
      static_cast<O*>(g.y)[n * g.ldo + v] = O(y);
    }
  }
}

}  // namespace nvs

struct NcbAdapterHead {
  int device = 0, dtype = 0, in = 0, out = 0, max_rows = 0, slots = 0, max_rank = 0, rpad = 0;
  std::mutex mu;
  void* mem = nullptr;
  void *a = nullptr, *b = nullptr;
  int32_t* ranks = nullptr;
  float *scales = nullptr, *u = nullptr;
  const void* w = nullptr;
  int64_t ldw = 0;
};

namespace {

struct AhDevice {  // the handle's device for the duration of a call
  int prev = -1;
  bool ok = false;
  explicit AhDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    ok = prev == dev || cudaSetDevice(dev) == cudaSuccess;
    if (prev == dev) prev = -1;
  }
  ~AhDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

bool ah_aligned(const void* p, uintptr_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

int ah_launched() { return cudaGetLastError() == cudaSuccess ? NCB_OK : NCB_ERROR_LAUNCH_FAILED; }

template <typename E>
int ah_pack(NcbAdapterHead* h, int slot, const void* a, int64_t lda, const void* b, int64_t ldb,
            int rank, float scale, cudaStream_t st) {
  nvs::adapter_pack_kernel<E><<<512, 256, 0, st>>>(
      static_cast<E*>(h->a), static_cast<E*>(h->b), h->ranks, h->scales, slot, h->in, h->out,
      h->rpad, static_cast<const E*>(a), lda, static_cast<const E*>(b), ldb, rank, scale);
  return ah_launched();
}

template <typename E>
int ah_project(const nvs::AhArgs& g, bool wide, cudaStream_t st) {
  if (g.ids) {
    const int64_t warps = (int64_t)g.rows * g.rpad;
    nvs::adapter_shrink_kernel<E><<<(unsigned)((warps + 7) / 8), 256, 0, st>>>(g);
  }
  const dim3 grid((g.out + 63) / 64, (g.rows + 63) / 64);
  if (wide) nvs::adapter_project_kernel<E, float><<<grid, 256, 0, st>>>(g);
  else nvs::adapter_project_kernel<E, E><<<grid, 256, 0, st>>>(g);
  return ah_launched();
}

}  // namespace

extern "C" {

NCB_API int ncb_adapter_head_create(int device, int dtype, int in_features, int out_features,
                                    int max_rows, int max_adapters, int max_rank,
                                    NcbAdapterHead** out) {
  if (!out) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  *out = nullptr;
  if (device < 0 || (dtype != NCB_DTYPE_F16 && dtype != NCB_DTYPE_BF16) || in_features <= 0 ||
      out_features <= 0 || max_rows <= 0 || max_adapters < 0 || max_rank < 0 ||
      (max_adapters > 0 && max_rank == 0))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (max_adapters > nvs::AH_MAX_ADAPTERS || max_rank > nvs::AH_MAX_RANK ||
      in_features > (1 << 20) || out_features > (1 << 24) || max_rows > (1 << 16))
    return ncb_record_status(NCB_ERROR_CAPACITY);
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || device >= count)
    return ncb_record_status(NCB_ERROR_NO_DEVICE);
  AhDevice guard(device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  NcbAdapterHead* h = new (std::nothrow) NcbAdapterHead();
  if (!h) return ncb_record_status(NCB_ERROR_ALLOC_FAILED);
  h->device = device;
  h->dtype = dtype;
  h->in = in_features;
  h->out = out_features;
  h->max_rows = max_rows;
  h->slots = max_adapters;
  h->max_rank = max_rank;
  h->rpad = (max_rank + 15) / 16 * 16;
  size_t off = 0;
  auto carve = [&](size_t bytes) {
    const size_t o = off;
    off += (bytes + 255) / 256 * 256;
    return o;
  };
  const size_t per = (size_t)h->slots * h->rpad;
  const size_t o_a = carve(per * h->in * 2), o_b = carve(per * h->out * 2);
  const size_t o_r = carve((size_t)h->slots * 4), o_s = carve((size_t)h->slots * 4);
  const size_t o_u = carve((size_t)max_rows * h->rpad * 4);
  if (cudaMalloc(&h->mem, off + 256) != cudaSuccess) {
    cudaGetLastError();
    delete h;
    return ncb_record_status(NCB_ERROR_ALLOC_FAILED);
  }
  char* m = static_cast<char*>(h->mem);
  h->a = m + o_a;
  h->b = m + o_b;
  h->ranks = reinterpret_cast<int32_t*>(m + o_r);
  h->scales = reinterpret_cast<float*>(m + o_s);
  h->u = reinterpret_cast<float*>(m + o_u);
  if (cudaMemset(h->ranks, 0, (size_t)h->slots * 4 + 4) != cudaSuccess ||
      cudaDeviceSynchronize() != cudaSuccess) {
    cudaFree(h->mem);
    delete h;
    return ncb_record_status(NCB_ERROR_INIT_FAILED);
  }
  *out = h;
  return ncb_record_status(NCB_OK);
}

NCB_API int ncb_adapter_head_destroy(NcbAdapterHead* h) {
  if (!h) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  {
    AhDevice guard(h->device);
    cudaDeviceSynchronize();
    cudaFree(h->mem);
  }
  delete h;
  return ncb_record_status(NCB_OK);
}

NCB_API int ncb_adapter_head_set_weight_device(NcbAdapterHead* h, const void* d_weight, int64_t ld,
                                               void* stream) {
  if (!h) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  (void)stream;
  if (!d_weight || ld < h->in || !ah_aligned(d_weight, 2))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  std::lock_guard<std::mutex> lk(h->mu);
  h->w = d_weight;
  h->ldw = ld;
  return ncb_record_status(NCB_OK);
}

NCB_API int ncb_adapter_head_set_adapter_device(NcbAdapterHead* h, int slot, const void* d_a,
                                                int64_t lda, const void* d_b, int64_t ldb,
                                                int rank, float scale, void* stream) {
  if (!h) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  if (slot < 0 || slot >= h->slots || rank <= 0 || !d_a || !d_b || lda < h->in || ldb < rank ||
      !std::isfinite(scale) || !ah_aligned(d_a, 2) || !ah_aligned(d_b, 2))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rank > h->max_rank) return ncb_record_status(NCB_ERROR_CAPACITY);
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return ncb_record_status(
      h->dtype == NCB_DTYPE_BF16
          ? ah_pack<__nv_bfloat16>(h, slot, d_a, lda, d_b, ldb, rank, scale, st)
          : ah_pack<__half>(h, slot, d_a, lda, d_b, ldb, rank, scale, st));
}

NCB_API int ncb_adapter_head_clear_adapter_device(NcbAdapterHead* h, int slot, void* stream) {
  if (!h) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  if (slot < 0 || slot >= h->slots) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  return ncb_record_status(cudaMemsetAsync(h->ranks + slot, 0, 4, static_cast<cudaStream_t>(stream)) ==
                                   cudaSuccess
                               ? NCB_OK
                               : NCB_ERROR_LAUNCH_FAILED);
}

NCB_API int ncb_adapter_head_project_device(NcbAdapterHead* h, const void* d_x, int64_t ldx,
                                            int rows, const int32_t* d_adapter_ids, void* d_out,
                                            int out_dtype, int64_t ldo, void* stream) {
  if (!h || !h->w) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  if (rows < 0 || (out_dtype != NCB_DTYPE_F32 && out_dtype != h->dtype))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows == 0) return ncb_record_status(NCB_OK);
  if (!d_x || !d_out || ldx < h->in || ldo < h->out || !ah_aligned(d_x, 2) ||
      !ah_aligned(d_out, out_dtype == NCB_DTYPE_F32 ? 4 : 2) || !ah_aligned(d_adapter_ids, 4))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows > h->max_rows) return ncb_record_status(NCB_ERROR_CAPACITY);
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  nvs::AhArgs g{};
  g.x = d_x;
  g.ldx = ldx;
  g.w = h->w;
  g.ldw = h->ldw;
  g.rows = rows;
  g.in = h->in;
  g.out = h->out;
  g.slots = h->slots;
  g.rpad = h->rpad;
  g.ids = h->slots ? d_adapter_ids : nullptr;
  g.a = h->a;
  g.b = h->b;
  g.ranks = h->ranks;
  g.scales = h->scales;
  g.u = h->u;
  g.y = d_out;
  g.ldo = ldo;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return ncb_record_status(h->dtype == NCB_DTYPE_BF16
                               ? ah_project<__nv_bfloat16>(g, out_dtype == NCB_DTYPE_F32, st)
                               : ah_project<__half>(g, out_dtype == NCB_DTYPE_F32, st));
}

}  // extern "C"
