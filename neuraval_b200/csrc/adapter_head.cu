// LM head with low-rank adapters of many requests (sm_100a):
//   out[n, :] = W x_n + scale_s B_s (A_s x_n),  s = adapter_ids[n].
//
// head_kernel multiplies on the tensor cores: 128 outputs (256 for a pair of CTAs)
// by a tile of NT <= 256 rows of the batch, the sums in TMEM. The weight is the
// 128-row operand, so a few rows waste no tensor-core rows and every weight byte is
// read once. The adapters are part of the same sums, a longer inner axis:
//   out^T += B_e U_e^T   for each entry e = (16 ranks of a slot, a block of rows),
// U_e holding u_n = scale_s A_s x_n for the rows n of the block that name the slot
// and zeros for the others, split into 16-bit values, each with its own product (one
// would round u to 8 bits of bf16): two, u = hi + lo, 16 bits, where the output is
// rounded to fewer anyway, and three for bf16 with an fp32 output (with two the
// result was 1.2e-6 off, more than all of the sums). fp16 has 22 bits in two, but none
// below 2^-24, so what is lost of a small u is 2^-25 instead; a third value would not
// change that, and B in a wider type would double its bytes and its products.
//
// Tiles of up to AH_SINGLE rows have one block, the tile. Larger tiles are sorted by
// slot first (adapter_sort_kernel copies x in that order) and cut into blocks of 32
// rows, so that a slot's entries cover little more than its own rows: with whole
// tiles as blocks, 32 slots of 16 ranks took a quarter of the tensor cores' time
// (256x4096x128256: 284 us, without adapters 234). The sort costs a launch that
// nothing hides. Single CTAs against pairs, 12 slots of 16 ranks (16 for 128 rows):
// 80x4096x128256 194 and 203 us, 96 rows 198 and 197 (fp32 207 and 223), 128 rows 217
// and 211; 96x2048x32000 40 and 46.
//
// adapter_shrink_kernel computes u while the head multiplies its first tile; the
// head waits for it only before the first entry (programmatic dependent launch).
//
// Up to about 256 rows the head is bound by the weight's bytes (32x4096x128256, 8
// slots of 16 ranks, fp32 output: 183 us in a short loop, 191 in a long one, 5.8 TB/s;
// without adapters 170), beyond by the tensor cores and the power they draw
// (512x4096x151936, 16 slots of 32 ranks: 636 us alone, 1.0 PFLOP/s, 748 us in a long
// loop whose clock sinks to 1 GHz; without adapters 474 and 576).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <new>
#include <type_traits>

#include "bounded_wait.cuh"
#include "navsampler.h"

int ncb_record_status(int st);

namespace nvs {

constexpr int AH_MAX_ADAPTERS = 1024;
constexpr int AH_MAX_RANK = 128;
constexpr int AH_BM = 128;        // outputs per tile
constexpr int AH_BK = 64;         // inner values per stage: 128-byte rows
constexpr int AH_NT = 256;        // rows of the batch per tile at most
constexpr int AH_A_BYTES = AH_BM * AH_BK * 2;
constexpr int AH_MAX_STAGES = 12;
constexpr int AH_SMEM = 208 * 1024;  // stages; leaves room for a shrink CTA on the SM
constexpr int AH_EPILOGUE = 8;    // warps that write results
constexpr int AH_THREADS = (AH_EPILOGUE + 2) * 32;  // and a copying and a multiplying one
constexpr int AH_PIECE = 8;       // stages added up in TMEM for an fp32 output
constexpr int AH_SINGLE = 96;     // rows per tile up to which single CTAs work, unsorted
constexpr int AH_BLOCK = 32;      // rows per block of larger tiles
constexpr int AH_PARTS = 3;       // 16-bit values that make up u, at most

// Adapter entries per stage. A stage, AH_A_BYTES + nh * 128 bytes, holds 4 KiB of B for
// each and, behind them, the entries' U, AH_PARTS * bh * 32 bytes each. (Copies cost
// about the same whatever their size, so pairs take four entries with one copy of U.)
constexpr int ah_per(int group) { return group == 2 ? 4 : 2; }
constexpr bool ah_fits(int group, int nh, int bh) {
  return ah_per(group) * (AH_BM * 32 + AH_PARTS * bh * 32) <= AH_A_BYTES + nh * 128;
}
// (single CTAs: bh = nh, and the entries' bytes grow by 192 nh, the stage's by 128 nh)
static_assert(ah_fits(1, AH_SINGLE, AH_SINGLE), "entries of a single CTA");
static_assert(ah_fits(2, (AH_SINGLE + 32) / 32 * 32 / 2, AH_BLOCK / 2), "entries of the smallest pair");

struct AhArgs {
  const void* x;
  int64_t ldx;
  int rows, in, kpad, out, slots, slices;  // slices: entries a slot can have
  int nt, nh, tiles_n;                     // rows per tile, of it per CTA, tiles of rows
  const int32_t* ids;
  const void* a;        // [slots][16 slices][kpad]
  int block, bh;        // rows per block, of it per CTA
  int parts, per;       // 16-bit values that make up u; entries per stage of the head
  void* x_sorted;       // [rows][kpad]
  int4* info;           // [tiles_n][AH_NT] by row: place, first entry, first and last place of its slot
  int32_t* order;       // [tiles_n][AH_NT] by place: row of the tile; NULL: as they come
  const int32_t* ranks; // per slot; 0: empty, < 0: |rank|, and B holds a non-finite value
  const float* scales;
  void* u;              // [tiles_n][block / bh][max_entries][parts][bh][16]
  int2* entries;        // [tiles_n][max_entries] slot * slices + slice, first place
  int32_t* counts;      // [tiles_n]
  int max_entries, opad;
  void* y;
  int64_t ldo;
  int share;   // outputs per CTA
  int groups;  // tiles of rows worked on at the same time, by neighbouring CTAs
  uint32_t idesc, idesc_u;
  int stages;
  uint32_t* error_word;  // in host memory
};

// ---- loading a slot ---------------------------------------------------------------
// Where value j of row r lies in a [rows][16] matrix as the tensor cores read it
// from shared memory (rows of 32 bytes, their halves swapped in every other group
// of four rows). B and U are kept like this in global memory, so that a tile of
// them is contiguous and is copied by rows of 512 bytes: TMA boxes of 32-byte rows
// took five times as long.
__host__ __device__ __forceinline__ int64_t ah_at(int64_t r, int j) {
  return r * 16 + (j ^ ((int)(r >> 2) & 1) << 3);
}

// B goes to [slice][outputs][16]: a 128-row tile of an entry is 4 KiB in a row. A
// value of B that is not finite would reach every row of a tile (0 times NaN);
// it is stored as 0 and the slot marked, and the slot's own rows come out as NaN.
template <typename E>
__global__ void adapter_pack_kernel(E* a, E* b, int32_t* ranks, int slot, int in, int kpad,
                                    int out, int opad, int slices, const E* sa,
                                    int64_t lda, const E* sb, int64_t ldb, int rank) {
  const int64_t na = (int64_t)slices * 16 * kpad, nb = (int64_t)slices * opad * 16;
  const int64_t t0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x, dt = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = t0; i < na; i += dt) {
    const int64_t j = i / kpad, k = i % kpad;
    a[slot * na + i] = j < rank && k < in ? sa[j * lda + k] : E(0.0f);
  }
  bool bad = false;
  for (int64_t i = t0; i < nb; i += dt) {
    const int64_t slice = i / ((int64_t)opad * 16), j = slice * 16 + i % 16, v = i / 16 % opad;
    E x = j < rank && v < out ? sb[v * ldb + j] : E(0.0f);
    if (!(fabsf((float)x) < INFINITY)) {
      bad = true;
      x = E(0.0f);
    }
    b[slot * nb + slice * opad * 16 + ah_at(v, (int)(i % 16))] = x;
  }
  if (bad) ranks[slot] = -rank;
}
__global__ void adapter_slot_kernel(int32_t* ranks, float* scales, int slot, int rank, float scale) {
  ranks[slot] = rank;
  scales[slot] = scale;
}

// x or the weight, copied to rows that start on 16-byte boundaries.
template <typename E>
__global__ void adapter_align_kernel(E* to, int64_t pitch, const E* from, int64_t ld, int64_t rows,
                                     int cols) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += blockDim.x) to[r * pitch + c] = from[r * ld + c];
}

// ---- u = scale A x --------------------------------------------------------------------
constexpr int AS_THREADS = 256;  // of the sort
constexpr int AU_THREADS = 128;  // of the shrink kernel
static_assert(AS_THREADS >= AH_NT && AS_THREADS * 4 == AH_MAX_ADAPTERS, "a row, four slots per thread");

template <typename E>
__device__ __forceinline__ float2 ah_pair(uint32_t w) {
  if constexpr (std::is_same_v<E, __nv_bfloat16>)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Eight values of a row of x from column k on; columns past the row are 0.
template <typename E>
__device__ __forceinline__ uint4 ah_row8(const E* row, int k, int in) {
  if (k + 8 <= in) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < in)
      w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[k + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Exclusive prefix over the CTA's threads; the sum of all to `total`.
__device__ __forceinline__ int as_scan(int v, int32_t* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int at = inc - v, all = 0;
#pragma unroll
  for (int w = 0; w < AS_THREADS / 32; ++w) {
    if (w < warp) at += warp_sum[w];
    all += warp_sum[w];
  }
  __syncthreads();
  *total = all;
  return at;
}
// The slot of a row of the batch, -1 for none; its entries per block to `n`.
__device__ __forceinline__ int as_slot(const AhArgs& g, int row, int* n) {
  const int s = row < g.rows ? g.ids[row] : -1;
  *n = s >= 0 && s < g.slots ? (abs(g.ranks[s]) + 15) / 16 : 0;
  return *n ? s : -1;
}

// Larger tiles: grid (nt, tiles_n). The rows of a tile in the order of their slots
// (rows without one last), a CTA for each row: it finds the row's place, copies its
// x there and notes where its slot's entries are; row 0's CTA writes the tile's
// list of entries down. A slot whose rows reach over several blocks has an entry
// for each.
__global__ void __launch_bounds__(AS_THREADS) adapter_sort_kernel(const AhArgs g) {
  __shared__ int32_t first[AH_MAX_ADAPTERS];  // rows per slot, then its first place
  __shared__ int32_t entry[AH_MAX_ADAPTERS];  // its first entry
  __shared__ int32_t warp_sum[AS_THREADS / 32];
  const int t = threadIdx.x, r = blockIdx.x, tile = blockIdx.y, n0 = tile * g.nt;
#pragma unroll
  for (int j = 0; j < 4; ++j) first[4 * t + j] = 0;
  int n, mine_n;
  const int s = as_slot(g, t < g.nt ? n0 + t : g.rows, &n), mine = as_slot(g, n0 + r, &mine_n);
  __syncthreads();
  if (s >= 0) atomicAdd(&first[s], 1);
  __syncthreads();
  int rows[4], sum = 0, named;
#pragma unroll
  for (int j = 0; j < 4; ++j) sum += rows[j] = first[4 * t + j];
  int at = as_scan(sum, warp_sum, &named), parts[4], slices[4], count;
  sum = 0;
#pragma unroll
  for (int j = 0, a = at; j < 4; ++j) {
    slices[j] = rows[j] ? (abs(g.ranks[4 * t + j]) + 15) / 16 : 0;
    parts[j] = rows[j] ? (a + rows[j] - 1) / AH_BLOCK - a / AH_BLOCK + 1 : 0;
    sum += slices[j] * parts[j];
    a += rows[j];
  }
  int e = as_scan(sum, warp_sum, &count);
  int2* entries = g.entries + (int64_t)tile * g.max_entries;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    first[4 * t + j] = at;
    entry[4 * t + j] = e;
    if (r == 0)
      for (int i = 0; i < slices[j]; ++i)
        for (int b = 0; b < parts[j]; ++b)
          entries[e + i * parts[j] + b] =
              make_int2((4 * t + j) * g.slices + i, (at / AH_BLOCK + b) * AH_BLOCK);
    at += rows[j];
    e += slices[j] * parts[j];
  }
  if (r == 0 && t == 0) g.counts[tile] = count;
  const bool here = t < g.nt && n0 + t < g.rows;
  const int before = __syncthreads_count(here && s == mine && t < r),
            equal = __syncthreads_count(here && s == mine);
  if (n0 + r >= g.rows) return;
  const int start = mine >= 0 ? first[mine] : named, place = start + before;
  if (t == 0) {
    g.order[tile * AH_NT + place] = r;
    g.info[tile * AH_NT + r] = make_int4(place, mine >= 0 ? entry[mine] : 0, start, start + equal - 1);
  }
  // values of 16 bits, whatever their type
  const uint16_t* x = static_cast<const uint16_t*>(g.x) + (int64_t)(n0 + r) * g.ldx;
  uint16_t* to = static_cast<uint16_t*>(g.x_sorted) + (int64_t)(n0 + place) * g.kpad;
  if ((reinterpret_cast<uintptr_t>(g.x) & 15) == 0 && g.ldx % 8 == 0) {
    for (int k = 8 * t; k < g.in; k += 8 * AS_THREADS)
      *reinterpret_cast<uint4*>(to + k) = ah_row8(x, k, g.in);
  } else {
    for (int k = t; k < g.in; k += AS_THREADS) to[k] = x[k];
  }
}

// grid (nt, tiles_n): a CTA for a row, its 16 ranks at a time, 8 columns per thread
// and turn, summed over the threads at the end. The operations are few (rows * rank
// * in); what counts is that the kernel ends while the head still multiplies its
// first tile, so it is spread over as many CTAs as there are rows, four to an SM:
// the head starts when all of them have. Unsorted (nt <= AH_SINGLE), every CTA
// lists its tile's entries for itself, in the order of the slots.
template <typename E, bool SORTED>
__global__ void __launch_bounds__(AU_THREADS, 4) adapter_shrink_kernel(const AhArgs g) {
  // sorted: the head starts when every CTA is here, and so after the sort's end
  if constexpr (SORTED) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ int32_t key[AH_SINGLE];  // slot << 8 | entries of each row, the largest number for none
  __shared__ float part[AU_THREADS / 32][16];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int r = blockIdx.x, tile = blockIdx.y, n0 = tile * g.nt;
  int mine;
  const int slot = as_slot(g, n0 + r, &mine);
  E* u = static_cast<E*>(g.u) + (int64_t)tile * g.max_entries * g.parts * g.block * 16;
  // an entry's share of the block that holds row `at`; each part is bh rows
  auto row_of = [&](int e, int at) {
    return u + ((int64_t)(at / g.bh) * g.max_entries + e) * g.parts * g.bh * 16;
  };
  auto clear = [&](int e, int at, int half) {  // the half of the row, in every part
    for (int p = 0; p < g.parts; ++p)
      *reinterpret_cast<uint4*>(row_of(e, at) + p * g.bh * 16 + at % g.bh * 16 + half * 8) =
          make_uint4(0, 0, 0, 0);
  };
  int own, next, place;  // the row's first entry, how far to the next 16 ranks', the row in it
  const E* x = static_cast<const E*>(g.x) + (int64_t)(n0 + r) * g.ldx;
  if constexpr (SORTED) {
    if (!mine) return;
    const int4 info = g.info[tile * AH_NT + r];
    const int b0 = info.z / AH_BLOCK, b1 = info.w / AH_BLOCK;
    next = b1 - b0 + 1;
    own = info.y + info.x / AH_BLOCK - b0;
    place = info.x % AH_BLOCK;
    x = static_cast<const E*>(g.x_sorted) + (int64_t)(n0 + info.x) * g.kpad;
    if (info.x == info.z)  // the slot's first row clears what is not the slot's
      for (int j = 0; j < mine; ++j) {
        const int front = info.z % AH_BLOCK, back = AH_BLOCK - 1 - info.w % AH_BLOCK;
        const int e = info.y + j * next;
        for (int i = t; i < 2 * front; i += AU_THREADS) clear(e, i >> 1, i & 1);
        for (int i = t; i < 2 * back; i += AU_THREADS)
          clear(e + b1 - b0, AH_BLOCK - back + (i >> 1), i & 1);
      }
  } else {
    const int none = 0x7FFFFFFF;
    int kt = none;
    if (t < g.nt) {
      int n;
      const int s = as_slot(g, n0 + t, &n);
      if (s >= 0) kt = s << 8 | n;
      key[t] = kt;
    }
    __syncthreads();
    bool leads = kt != none;  // the slot's first row speaks for it
    for (int i = 0; leads && i < t; ++i) leads = key[i] != kt;
    __syncthreads();
    if (t < g.nt && !leads) key[t] = none;
    __syncthreads();
    // a slot's entries are behind those of all lower slots
    const int k = mine ? slot << 8 | mine : none;
    int before = 0, count = 0, mine_at = 0;
    for (int i = 0; i < g.nt; ++i) {
      const int ki = key[i], n = ki == none ? 0 : ki & 255;
      count += n;
      before += ki < k ? n : 0;
      mine_at += ki < kt ? n : 0;
    }
    own = before;
    next = 1;
    place = r;
    if (r == 0) {  // row 0's CTA writes the list down
      int2* entries = g.entries + (int64_t)tile * g.max_entries;
      if (leads)
        for (int i = 0; i < (kt & 255); ++i)
          entries[mine_at + i] = make_int2((kt >> 8) * g.slices + i, 0);
      if (t == 0) g.counts[tile] = count;
    }
    for (int i = t; i < 2 * count; i += AU_THREADS)
      if (i >> 1 < own || i >> 1 >= own + mine) clear(i >> 1, r, i & 1);
    if (!mine) return;
  }
  for (int slice = 0; slice < mine; ++slice) {
  float acc[16] = {};
  const E* a = static_cast<const E*>(g.a) + ((int64_t)slot * g.slices + slice) * 16 * (int64_t)g.kpad;
  for (int k = t * 8; k < g.kpad; k += AU_THREADS * 8) {
    const uint4 xv = ah_row8(x, k, g.in);
    uint4 av[16];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      av[j] = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)j * g.kpad + k));
    const float2 x0 = ah_pair<E>(xv.x), x1 = ah_pair<E>(xv.y), x2 = ah_pair<E>(xv.z),
                 x3 = ah_pair<E>(xv.w);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 a0 = ah_pair<E>(av[j].x), a1 = ah_pair<E>(av[j].y), a2 = ah_pair<E>(av[j].z),
                   a3 = ah_pair<E>(av[j].w);
      acc[j] = fmaf(a0.x, x0.x, fmaf(a0.y, x0.y, acc[j]));
      acc[j] = fmaf(a1.x, x1.x, fmaf(a1.y, x1.y, acc[j]));
      acc[j] = fmaf(a2.x, x2.x, fmaf(a2.y, x2.y, acc[j]));
      acc[j] = fmaf(a3.x, x3.x, fmaf(a3.y, x3.y, acc[j]));
    }
  }
  // sums over the warp: lane l ends with those of rank l / 2
#pragma unroll
  for (int half = 8, o = 16; half > 0; half >>= 1, o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float send = upper ? acc[j] : acc[j + half], keep = upper ? acc[j + half] : acc[j];
      acc[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 1);
  if ((lane & 1) == 0) part[warp][lane >> 1] = acc[0];
  __syncthreads();

  if (t < 16) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < AU_THREADS / 32; ++w) v += part[w][t];
    v *= g.scales[slot];
    E hi = E(v);
    if (g.ranks[slot] < 0 || !(fabsf((float)hi) < INFINITY)) hi = E(NAN);
    E* to = row_of(own + slice * next, place) + ah_at(place % g.bh, t);
    for (int p = 0; p < g.parts; ++p) {  // what the parts before have left, rounded
      to[(int64_t)p * g.bh * 16] = hi;
      v -= (float)hi;
      hi = E(v);
    }
  }
  __syncthreads();
  }
}

// ---- the product ------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ah_smem(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
// Every wait ends: after 2 s it gives up.
__device__ __forceinline__ bool ah_wait(uint32_t bar, uint32_t parity) {
  return wait_for(bar, parity, 1000000000u);
}
// A wait gave up: a word in host memory, which the handle's calls look at.
__device__ __forceinline__ void ah_failed(uint32_t* word, uint32_t where) {
  *(volatile uint32_t*)word = where;
  __threadfence_system();
}
__device__ __forceinline__ void ah_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// Shared addresses of a pair's CTAs differ in bit 24: without it, the first one's.
constexpr uint32_t AH_FIRST = 0xFEFFFFFFu;
template <int CG>
__device__ __forceinline__ void ah_arrive_first(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n"
        " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}" ::"r"(bar)
        : "memory");
}
// Copies into this CTA's own shared memory; in a pair the first CTA's barrier
// counts the bytes of both.
template <int CG>
__device__ __forceinline__ void ah_copy(uint32_t to, const CUtensorMap* map, uint32_t bar, int x,
                                         int y) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
            "r"(to),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
            "r"(to),
        "l"(map), "r"(bar & AH_FIRST), "r"(x), "r"(y)
        : "memory");
}
// Shared-memory operand whose rows of `span` bytes (32 or 128) lie one behind the
// other in the TMA's swizzle of that span, eight rows to a group.
__device__ __forceinline__ uint64_t ah_operand(uint32_t addr, int span) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(span * 8 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)(span == 128 ? 2 : 6) << 61;
}
template <int CG>
__device__ __forceinline__ void ah_multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc,
                                            bool add) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// The barrier (of both CTAs of a pair) is arrived at when the products issued so
// far have ended.
template <int CG>
__device__ __forceinline__ void ah_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::
            "r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void ah_all_sync() {
  if constexpr (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

__device__ __forceinline__ void ah_load16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// One CTA per SM, or (CG = 2) a pair of CTAs on two SMs whose tensor cores work on
// one product: each holds its own 128 outputs and half of the rows of x, and reads
// the other half from its neighbour.
//
// The outputs are dealt out evenly: every CTA takes g.share of them, a multiple of
// 16, in tiles of 128 and a last, lower one, so that all read the same number of
// weight bytes (whole tiles would leave a sixth of the SMs idle at 250 tiles). With
// several tiles of rows, neighbouring CTAs (or pairs) work on the same outputs with
// different ones of them, g.groups at a time, so that one reads from L2 what the
// other brought there: 148 CTAs' tiles of 1 MB would not stay in L2 until a CTA
// comes back to them (512x4096x75776 read its weight twice).
//
// CPT > 0 (fp32 output): the sum over the inner axis is cut into pieces of
// AH_PIECE stages, each summed in TMEM from zero and added up in registers, CPT
// columns of the batch per thread. The tensor cores truncate their sums, an error
// that grows with the number of additions: 256 in a row (4096 values) measured
// 3.9e-6 of the result, eight pieces of 32 a sixth of that. A 16-bit output's own
// rounding hides it, so there the sum is one piece.
template <typename O, int CG, int CPT>
__global__ void __launch_bounds__(AH_THREADS, 1)
    head_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_low,
                const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_u, const AhArgs g) {
  extern __shared__ uint8_t ah_raw[];
  __shared__ uint64_t bars[2 * AH_MAX_STAGES + 4];
  __shared__ uint32_t s_tmem;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int rank = CG == 1 ? 0 : (int)(blockIdx.x & 1);  // in the pair
  const uint32_t stage0 = (ah_smem(ah_raw) + 1023) & ~1023u;
  const int nh = g.nh;  // rows of x in this CTA
  const uint32_t stage_bytes = AH_A_BYTES + nh * 128;
  const uint32_t full = ah_smem(bars), empty = full + 8 * AH_MAX_STAGES,
                 done = empty + 8 * AH_MAX_STAGES, drained = done + 16;
  uint32_t columns = 32;
  while (columns < 2u * g.nt) columns *= 2;
  if (warp == AH_EPILOGUE + 1) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       ah_smem(&s_tmem)),
                   "r"(columns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       ah_smem(&s_tmem)),
                   "r"(columns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  if (t == 0) {
    for (int i = 0; i < AH_MAX_STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8 * i) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty + 8 * i) : "memory");
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(done + 8 * i) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(drained + 8 * i),
                   "r"(AH_EPILOGUE * CG)
                   : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  ah_all_sync<CG>();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const int steps = (g.in + AH_BK - 1) / AH_BK;
  const int piece = CPT ? AH_PIECE : steps;  // stages added up in TMEM
  const int pieces = (steps + piece - 1) / piece;
  const int at = blockIdx.x / CG, group = at % g.groups;
  const int v_begin = (at / g.groups * CG + rank) * g.share, tiles_m = (g.share + AH_BM - 1) / AH_BM;
  const int tiles_n = (g.tiles_n - group + g.groups - 1) / g.groups;  // this CTA's

  if (warp == AH_EPILOGUE) {  // ---- copies: the warp waits together, a lane issues ------------
    int s = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true, waited = false;
    if (g.order) asm volatile("fence.proxy.async.global;" ::: "memory");  // the sorted x
    for (int i = 0; ok && i < tiles_m * tiles_n; ++i) {
      const int m = i / tiles_n, n = group + i % tiles_n * g.groups;
      const int v0 = v_begin + m * AH_BM, high = min(AH_BM, g.share - m * AH_BM);
      const int2* entries = g.entries + (int64_t)n * g.max_entries;
      int count = 0;  // entries of the tile of rows; lane l holds the l-th of 32
      int2 mine{};
      if (waited && g.ids) {
        count = __ldcg(g.counts + n);
        if (lane < count) mine = __ldcg(entries + lane);
      }
      for (int k = 0; k < steps; ++k) {
        if (!(ok = ah_wait(empty + 8 * s, phase ^ 1))) break;
        if (lane == 0) {
          const uint32_t a = stage0 + s * stage_bytes, bar = full + 8 * s;
          if (rank == 0) ah_expect(bar, CG * (high * 128 + nh * 128));
          ah_copy<CG>(a, high == AH_BM ? &map_w : &map_low, bar, k * AH_BK, v0);
          ah_copy<CG>(a + AH_A_BYTES, &map_x, bar, k * AH_BK, n * g.nt + rank * nh);
        }
        __syncwarp();
        ++issued;
        if (++s == g.stages) s = 0, phase ^= 1;
      }
      if (!ok) break;
      if (!waited) {  // what follows reads the shrink kernel's results
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("fence.proxy.async.global;" ::: "memory");
        waited = true;
        if (g.ids) {
          count = __ldcg(g.counts + n);
          if (lane < count) mine = __ldcg(entries + lane);
        }
      }
      for (int e = 0; e < count; e += g.per) {
        if (e && (e & 31) == 0 && e + lane < count) mine = __ldcg(entries + e + lane);
        if (!(ok = ah_wait(empty + 8 * s, phase ^ 1))) break;
        const int several = min(g.per, count - e);
        const uint32_t a = stage0 + s * stage_bytes, bar = full + 8 * s;
        if (lane == 0) {  // U of a whole stage at once, whether it is full or not
          if (rank == 0) ah_expect(bar, CG * (several * AH_BM * 32 + g.per * g.parts * g.bh * 32));
          ah_copy<CG>(a + g.per * AH_BM * 32, &map_u, bar, 0,
                      (int)(((int64_t)(n * CG + rank) * g.max_entries + e) * g.parts * g.bh / 16));
        }
        for (int j = 0; j < several; ++j) {
          const int z = __shfl_sync(0xffffffffu, mine.x, (e & 31) + j);
          if (lane == 0)
            ah_copy<CG>(a + j * AH_BM * 32, &map_b, bar, 0, (int)(((int64_t)z * g.opad + v0) / 16));
        }
        __syncwarp();
        ++issued;
        if (++s == g.stages) s = 0, phase ^= 1;
      }
    }
    if (!ok) {  // gave up: no copy may be in flight when the CTA ends
      if (lane == 0) ah_failed(g.error_word, 1u);
      for (int i = 0; rank == 0 && i < g.stages && i < issued; ++i) {
        if (s-- == 0) s = g.stages - 1, phase ^= 1;
        ah_wait(full + 8 * s, phase);
      }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
  } else if (warp == AH_EPILOGUE + 1) {
    if (rank == 0) {  // ---- products: the warp waits together, a lane issues -------------------
      int s = 0, turn = 0;
      uint32_t phase = 0;
      bool ok = true, waited = false;
      for (int i = 0; ok && i < tiles_m * tiles_n; ++i) {
        const int n = group + i % tiles_n * g.groups;
        const int2* entries = g.entries + (int64_t)n * g.max_entries;
        int count = 0, mine = 0;  // as above; of an entry, the first place of its block
        if (waited && g.ids) {
          count = __ldcg(g.counts + n);
          if (lane < count) mine = __ldcg(&entries[lane].y);
        }
        for (int q = 0; ok && q < pieces; ++q, ++turn) {
          const uint32_t acc = tmem + (turn & 1) * g.nt;
          if (!(ok = ah_wait(drained + 8 * (turn & 1), ((turn >> 1) & 1) ^ 1))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int here = min(piece, steps - q * piece);
          for (int k = 0; k < here; ++k) {
            if (!(ok = ah_wait(full + 8 * s, phase))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (lane == 0) {
              const uint64_t a = ah_operand(stage0 + s * stage_bytes, 128);
              const uint64_t b = ah_operand(stage0 + s * stage_bytes + AH_A_BYTES, 128);
#pragma unroll
              for (int j = 0; j < AH_BK / 16; ++j)
                ah_multiply<CG>(acc, a + 2 * j, b + 2 * j, g.idesc, (k | j) != 0);
              ah_commit<CG>(empty + 8 * s);
            }
            __syncwarp();
            if (++s == g.stages) s = 0, phase ^= 1;
          }
          if (!ok) break;
          if (q == pieces - 1) {  // the adapters
            if (!waited) {
              asm volatile("griddepcontrol.wait;" ::: "memory");
              waited = true;
              if (g.ids) {
                count = __ldcg(g.counts + n);
                if (lane < count) mine = __ldcg(&entries[lane].y);
              }
            }
            for (int e = 0; e < count; e += g.per) {
              if (e && (e & 31) == 0 && e + lane < count) mine = __ldcg(&entries[e + lane].y);
              if (!(ok = ah_wait(full + 8 * s, phase))) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              const int several = min(g.per, count - e);
              const uint32_t base = stage0 + s * stage_bytes;
              for (int j = 0; j < several; ++j) {
                const int place = __shfl_sync(0xffffffffu, mine, (e & 31) + j);
                if (lane == 0) {
                  const uint64_t a = ah_operand(base + j * AH_BM * 32, 32);
                  for (int p = 0; p < g.parts; ++p)
                    ah_multiply<CG>(acc + place, a,
                                    ah_operand(base + g.per * AH_BM * 32 + (j * g.parts + p) * g.bh * 32, 32),
                                    g.idesc_u, true);
                }
              }
              if (lane == 0) ah_commit<CG>(empty + 8 * s);
              __syncwarp();
              if (++s == g.stages) s = 0, phase ^= 1;
            }
            if (!ok) break;
          }
          if (lane == 0) ah_commit<CG>(done + 8 * (turn & 1));
          __syncwarp();
        }
      }
      if (!ok) {
        // products in flight end before TMEM is given back
        if (lane == 0) {
          ah_failed(g.error_word, 2u);
          ah_commit<CG>(done + 8 * (turn & 1));
        }
        ah_wait(done + 8 * (turn & 1), (turn >> 1) & 1);
      }
    }
  } else {  // ---- results: warp w reads the 32 outputs of its quarter of TMEM, half of the rows --
    if (g.order) asm volatile("griddepcontrol.wait;" ::: "memory");
    int turn = 0;
    bool ok = true;
    O* y = static_cast<O*>(g.y);
    const int half = (g.nt / 2 + 15) / 16 * 16, c_begin = (warp >> 2) * half,
              c_end = min(g.nt, c_begin + half);
    for (int i = 0; ok && i < tiles_m * tiles_n; ++i) {
      const int m = i / tiles_n, n = group + i % tiles_n * g.groups, n0 = n * g.nt;
      const int in_tile = (warp & 3) * 32 + lane, v = v_begin + m * AH_BM + in_tile;
      const bool store = v < g.out && m * AH_BM + in_tile < g.share;
      const int here = min(c_end, g.rows - n0);  // columns with a row behind them end here
      O* to = y + (int64_t)n0 * g.ldo + v;
      const int32_t* order = g.order + n * AH_NT;
      auto put = [&](int c, float x) {  // the row in place c of the tile
        if (c < here) to[(int64_t)(g.order ? order[c] : c) * g.ldo] = O(x);
      };
      if constexpr (CPT > 0) {
        float sum[CPT];
#pragma unroll
        for (int c = 0; c < CPT; ++c) sum[c] = 0.0f;
        for (int q = 0; q < pieces; ++q, ++turn) {
          if (!(ok = ah_wait(done + 8 * (turn & 1), (turn >> 1) & 1))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t acc = tmem + (turn & 1) * g.nt + ((uint32_t)(warp & 3) << 21) + c_begin;
#pragma unroll
          for (int c = 0; c < CPT; c += 16)
            if (c_begin + c < here) {
              uint32_t r[16];
              ah_load16(acc + c, r);
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(r[j]);
            }
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) ah_arrive_first<CG>(drained + 8 * (turn & 1));
        }
        if (ok && store) {
#pragma unroll
          for (int c = 0; c < CPT; ++c) put(c_begin + c, sum[c]);
        }
      } else {
        if (!(ok = ah_wait(done + 8 * (turn & 1), (turn >> 1) & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + (turn & 1) * g.nt + ((uint32_t)(warp & 3) << 21);
        for (int c = c_begin; c < here; c += 16) {
          uint32_t r[16];
          ah_load16(acc + c, r);
          if (store) {
#pragma unroll
            for (int j = 0; j < 16; ++j) put(c + j, __uint_as_float(r[j]));
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) ah_arrive_first<CG>(drained + 8 * (turn & 1));
        ++turn;
      }
    }
    if (!ok && t == 0) ah_failed(g.error_word, 4u);
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  ah_all_sync<CG>();  // neither CTA of a pair ends while the other may still arrive in it
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == AH_EPILOGUE + 1) {
    if constexpr (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
  }
}

}  // namespace nvs

struct NcbAdapterHead {
  int device = 0, dtype = 0, in = 0, kpad = 0, out = 0, max_rows = 0, slots = 0, max_rank = 0;
  int slices = 0, num_sms = 0;
  int opad = 0;   // outputs, a multiple of 16
  int share = 0;  // outputs of a CTA: the same number for each, a multiple of 16
  std::mutex mu;
  void* mem = nullptr;  // everything below but the error word, w and w_own
  void *a = nullptr, *b = nullptr, *u = nullptr, *x_own = nullptr;
  int32_t *ranks = nullptr, *counts = nullptr, *order = nullptr;
  int2* entries = nullptr;
  int4* info = nullptr;
  float* scales = nullptr;
  uint32_t* error_word = nullptr;  // pinned: not 0 once a wait in a kernel has given up
  void* w_own = nullptr;  // the weight's copy, where it cannot be read in place
  bool has_w = false;
  const void* w = nullptr;  // what is read: the caller's weight or the copy
  int64_t ldw = 0;
  CUtensorMap map_w{}, map_low{}, map_b{};  // map_low: a CTA's last, lower tile
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
bool ah_gave_up(const NcbAdapterHead* h) {
  return *static_cast<const volatile uint32_t*>(h->error_word) != 0;
}
int ah_launched() { return cudaGetLastError() == cudaSuccess ? NCB_OK : NCB_ERROR_LAUNCH_FAILED; }

using AhEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
AhEncode ah_encode() {
  static const AhEncode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<AhEncode>(p);
  }();
  return fn;
}
// A map of a matrix of 16-bit values, rows ld apart, read by boxes.
bool ah_map(CUtensorMap* map, int dtype, const void* base, int64_t cols, int64_t rows, int64_t ld,
             int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const AhEncode fn = ah_encode();
  return fn && fn(map, dtype == NCB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  2, const_cast<void*>(base), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Whether a matrix of 16-bit values can be read by tiles in place.
bool ah_readable(const void* p, int64_t ld) { return ah_aligned(p, 16) && ld % 8 == 0; }

template <typename E>
int ah_pack(NcbAdapterHead* h, int slot, const void* a, int64_t lda, const void* b, int64_t ldb,
            int rank, float scale, cudaStream_t st) {
  nvs::adapter_slot_kernel<<<1, 1, 0, st>>>(h->ranks, h->scales, slot, rank, scale);
  nvs::adapter_pack_kernel<E><<<4 * h->num_sms, 256, 0, st>>>(
      static_cast<E*>(h->a), static_cast<E*>(h->b), h->ranks, slot, h->in, h->kpad,
      h->out, h->opad, h->slices, static_cast<const E*>(a), lda, static_cast<const E*>(b), ldb, rank);
  return ah_launched();
}

void ah_align(void* to, int64_t pitch, const void* from, int64_t ld, int64_t rows, int cols,
              int num_sms, cudaStream_t st) {
  const int64_t most = 8LL * num_sms;
  nvs::adapter_align_kernel<uint16_t><<<(unsigned)(rows < most ? rows : most), 256, 0, st>>>(
      static_cast<uint16_t*>(to), pitch, static_cast<const uint16_t*>(from), ld, rows, cols);
}

constexpr int64_t AH_L2 = 64ll << 20;  // of 126 MB: what weight tiles may take of it

struct AhMaps {
  CUtensorMap w, low, x, b, u;
};

// `beside`: it may start while the kernel before it still runs, and waits for that
// one itself.
template <typename... A>
bool ah_start(void (*kernel)(A...), dim3 grid, int threads, size_t smem, int cluster, bool beside,
              cudaStream_t st, const std::common_type_t<A>&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = beside ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess;
}

template <typename O, int CG, int CPT>
bool ah_launch(const AhMaps& m, const nvs::AhArgs& g, cudaStream_t st) {
  const int units = ((g.out + g.share - 1) / g.share + CG - 1) / CG;  // CTAs or pairs with outputs
  return ah_start(nvs::head_kernel<O, CG, CPT>, dim3(units * g.groups * CG), nvs::AH_THREADS,
                  (size_t)g.stages * (nvs::AH_A_BYTES + g.nh * 128) + 1024, CG, g.ids != nullptr, st,
                  m.w, m.low, m.x, m.b, m.u, g);
}
template <typename E, int CG>
int ah_head(const AhMaps& m, const nvs::AhArgs& g, bool wide, cudaStream_t st) {
  bool ok = true;
  if (g.ids) {
    const dim3 grid(g.nt, g.tiles_n);
    if constexpr (CG == 2)
      ok = ah_start(nvs::adapter_sort_kernel, grid, nvs::AS_THREADS, 0, 1, false, st, g);
    ok = ok && ah_start(nvs::adapter_shrink_kernel<E, CG == 2>, grid, nvs::AU_THREADS, 0, 1, CG == 2, st, g);
  }
  // fp32 sums stay in registers: those of half of the tile's rows per thread
  if (!wide) ok = ok && ah_launch<E, CG, 0>(m, g, st);
  else if constexpr (CG == 1)
    ok = ok && (g.nt <= 32 ? ah_launch<float, 1, 16>(m, g, st) : ah_launch<float, 1, 64>(m, g, st));
  else
    ok = ok && (g.nt <= 128 ? ah_launch<float, 2, 64>(m, g, st) : ah_launch<float, 2, 128>(m, g, st));
  return ok ? NCB_OK : NCB_ERROR_LAUNCH_FAILED;
}

// The shrink kernel asks for the shared-memory split that the head needs: an SM
// changes it only when it is idle, and the two are to run side by side.
bool ah_share() {
  for (const void* fn : {(const void*)nvs::adapter_sort_kernel,
                         (const void*)nvs::adapter_shrink_kernel<__nv_bfloat16, false>,
                         (const void*)nvs::adapter_shrink_kernel<__nv_bfloat16, true>,
                         (const void*)nvs::adapter_shrink_kernel<__half, false>,
                         (const void*)nvs::adapter_shrink_kernel<__half, true>})
    if (cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared) != cudaSuccess)
      return false;
  return true;
}
bool ah_raise() {
  for (const void* fn :
       {(const void*)nvs::head_kernel<__nv_bfloat16, 1, 0>, (const void*)nvs::head_kernel<__nv_bfloat16, 2, 0>,
        (const void*)nvs::head_kernel<__half, 1, 0>, (const void*)nvs::head_kernel<__half, 2, 0>,
        (const void*)nvs::head_kernel<float, 1, 16>, (const void*)nvs::head_kernel<float, 1, 64>,
        (const void*)nvs::head_kernel<float, 2, 64>, (const void*)nvs::head_kernel<float, 2, 128>})
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, nvs::AH_SMEM + 1024) !=
        cudaSuccess)
      return false;
  return true;
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
  h->slices = (max_rank + 15) / 16;
  h->opad = (out_features + 15) / 16 * 16;
  h->kpad = (in_features + nvs::AH_BK - 1) / nvs::AH_BK * nvs::AH_BK;
  cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device);
  const int ctas = h->num_sms / 2 * 2;  // whole pairs
  h->share = ((h->out + ctas - 1) / ctas + 15) / 16 * 16;
  size_t off = 0;
  auto carve = [&](size_t bytes) {
    const size_t o = off;
    off += (bytes + 255) / 256 * 256;
    return o;
  };
  const size_t tiles = ((size_t)max_rows + nvs::AH_NT - 1) / nvs::AH_NT;
  // entries of a tile: a block for each of its slots' 16 ranks, and one more for each
  // border between blocks that a slot's rows reach over
  const size_t most = h->slots ? ((size_t)(h->slots < nvs::AH_NT ? h->slots : nvs::AH_NT) +
                                  nvs::AH_NT / nvs::AH_BLOCK) * h->slices : 0;
  const size_t per = (size_t)h->slots * h->slices * 16;
  const size_t o_a = carve(per * h->kpad * 2), o_b = carve(per * h->opad * 2);
  const size_t o_x = carve((size_t)max_rows * h->kpad * 2);
  const size_t o_u = carve(tiles * most * nvs::AH_PARTS * nvs::AH_SINGLE * 16 * 2);  // the larger block
  const size_t o_e = carve(tiles * most * sizeof(int2)), o_c = carve(tiles * 4);
  const size_t o_i = carve(tiles * nvs::AH_NT * sizeof(int4)), o_o = carve(tiles * nvs::AH_NT * 4);
  const size_t o_s = carve((size_t)h->slots * 4), o_r = carve((size_t)h->slots * 4);
  if (cudaMalloc(&h->mem, off) != cudaSuccess ||
      cudaHostAlloc(&h->error_word, sizeof(uint32_t), cudaHostAllocMapped) != cudaSuccess) {
    cudaGetLastError();
    cudaFree(h->mem);
    delete h;
    return ncb_record_status(NCB_ERROR_ALLOC_FAILED);
  }
  *h->error_word = 0;
  char* m = static_cast<char*>(h->mem);
  h->a = m + o_a;
  h->b = m + o_b;
  h->x_own = m + o_x;
  h->u = m + o_u;
  h->entries = reinterpret_cast<int2*>(m + o_e);
  h->info = reinterpret_cast<int4*>(m + o_i);
  h->order = reinterpret_cast<int32_t*>(m + o_o);
  h->counts = reinterpret_cast<int32_t*>(m + o_c);
  h->scales = reinterpret_cast<float*>(m + o_s);
  h->ranks = reinterpret_cast<int32_t*>(m + o_r);
  bool ok = ah_share() && ah_raise() &&
            (!h->slots || cudaMemset(h->ranks, 0, (size_t)h->slots * 4) == cudaSuccess) &&
            cudaDeviceSynchronize() == cudaSuccess;
  if (ok && h->slots)  // 16 rows of 16 values are a row of the map
    ok = ah_map(&h->map_b, dtype, h->b, 256, (int64_t)per * h->opad / 256, 256, 256,
                 nvs::AH_BM / 16, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!ok) {
    cudaGetLastError();
    cudaFree(h->mem);
    cudaFreeHost(h->error_word);
    delete h;
    return ncb_record_status(NCB_ERROR_INIT_FAILED);
  }
  *out = h;
  return ncb_record_status(NCB_OK);
}

NCB_API int ncb_adapter_head_destroy(NcbAdapterHead* h) {
  if (!h) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  bool error = false;
  {
    AhDevice guard(h->device);
    error = cudaDeviceSynchronize() != cudaSuccess || ah_gave_up(h);
    cudaFree(h->mem);
    cudaFree(h->w_own);
    cudaFreeHost(h->error_word);
  }
  delete h;
  return ncb_record_status(error ? NCB_ERROR_LAUNCH_FAILED : NCB_OK);
}

NCB_API int ncb_adapter_head_status(NcbAdapterHead* h) {
  if (!h) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  return ncb_record_status(ah_gave_up(h) ? NCB_ERROR_LAUNCH_FAILED : NCB_OK);
}

NCB_API int ncb_adapter_head_set_weight_device(NcbAdapterHead* h, const void* d_weight, int64_t ld,
                                               void* stream) {
  if (!h) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  if (!d_weight || ld < h->in || !ah_aligned(d_weight, 2))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  if (!ah_readable(d_weight, ld)) {
    if (!h->w_own && cudaMalloc(&h->w_own, (size_t)h->out * h->kpad * 2) != cudaSuccess) {
      cudaGetLastError();
      h->w_own = nullptr;
      return ncb_record_status(NCB_ERROR_ALLOC_FAILED);
    }
    ah_align(h->w_own, h->kpad, d_weight, ld, h->out, h->in, h->num_sms,
             static_cast<cudaStream_t>(stream));
    if (ah_launched() != NCB_OK) return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
    d_weight = h->w_own;
    ld = h->kpad;
  }
  h->w = d_weight;
  h->ldw = ld;
  h->has_w = ah_map(&h->map_w, h->dtype, d_weight, h->in, h->out, ld, nvs::AH_BK, nvs::AH_BM,
                     CU_TENSOR_MAP_SWIZZLE_128B) &&
             ah_map(&h->map_low, h->dtype, d_weight, h->in, h->out, ld, nvs::AH_BK,
                     (h->share - 1) % nvs::AH_BM + 1, CU_TENSOR_MAP_SWIZZLE_128B);
  return ncb_record_status(h->has_w ? NCB_OK : NCB_ERROR_INIT_FAILED);
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
  if (!h || !h->has_w) return ncb_record_status(NCB_ERROR_NOT_INITIALIZED);
  if (rows < 0 || (out_dtype != NCB_DTYPE_F32 && out_dtype != h->dtype))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows == 0) return ncb_record_status(NCB_OK);
  if (!d_x || !d_out || ldx < h->in || ldo < h->out || !ah_aligned(d_x, 2) ||
      !ah_aligned(d_out, out_dtype == NCB_DTYPE_F32 ? 4 : 2) || !ah_aligned(d_adapter_ids, 4))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows > h->max_rows) return ncb_record_status(NCB_ERROR_CAPACITY);
  if (ah_gave_up(h)) return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  nvs::AhArgs g{};
  g.rows = rows;
  g.in = h->in;
  g.kpad = h->kpad;
  g.out = h->out;
  g.opad = h->opad;
  g.slots = h->slots;
  g.slices = h->slices;
  // tiles of up to 256 rows, all of one size; pairs of CTAs where they are large
  g.tiles_n = (rows + nvs::AH_NT - 1) / nvs::AH_NT;
  const int tile = (rows + g.tiles_n - 1) / g.tiles_n;
  const int group = tile > nvs::AH_SINGLE ? 2 : 1;
  g.nt = (tile + 16 * group - 1) / (16 * group) * (16 * group);
  g.nh = g.nt / group;
  g.ids = h->slots ? d_adapter_ids : nullptr;
  const bool sorted = g.ids && group == 2;
  g.block = group == 2 ? nvs::AH_BLOCK : g.nt;
  g.bh = g.block / group;
  g.parts = h->dtype == NCB_DTYPE_BF16 && out_dtype == NCB_DTYPE_F32 ? nvs::AH_PARTS : 2;
  g.per = nvs::ah_per(group);
  g.max_entries = (h->slots < nvs::AH_NT ? h->slots : nvs::AH_NT) * h->slices +
                  nvs::AH_NT / nvs::AH_BLOCK * h->slices;
  g.a = h->a;
  g.ranks = h->ranks;
  g.scales = h->scales;
  g.u = h->u;
  g.entries = h->entries;
  g.counts = h->counts;
  g.info = h->info;
  g.order = sorted ? h->order : nullptr;
  g.x_sorted = h->x_own;
  g.y = d_out;
  g.ldo = ldo;
  // fp32 sums, both operands of the head's type with the inner axis in rows
  const uint32_t type = h->dtype == NCB_DTYPE_BF16 ? 1u : 0u;
  const uint32_t kind = 1u << 4 | type << 7 | type << 10 | (uint32_t)(group * nvs::AH_BM / 16) << 24;
  g.idesc = kind | (uint32_t)(g.nt / 8) << 17;
  g.idesc_u = kind | (uint32_t)(g.block / 8) << 17;
  const int stage = nvs::AH_A_BYTES + g.nh * 128;
  g.stages = nvs::AH_SMEM / stage < nvs::AH_MAX_STAGES ? nvs::AH_SMEM / stage : nvs::AH_MAX_STAGES;
  // Tiles of rows at the same time: as many as take the fewest turns (tiles of
  // outputs times tiles of rows, of one CTA), among those whose weight tiles stay in
  // L2 until the CTA comes back to them, or that come back to none.
  g.share = h->share;
  g.groups = 1;
  int64_t turns = INT64_MAX;
  for (int n = 1; n <= g.tiles_n && n <= 8; ++n) {
    const int ctas = h->num_sms / group / n * group;
    const int share = ((h->out + ctas - 1) / ctas + 15) / 16 * 16;
    const int64_t live = (int64_t)ctas * nvs::AH_BM * h->kpad * 2;
    const int64_t t = (int64_t)((share + nvs::AH_BM - 1) / nvs::AH_BM) * ((g.tiles_n + n - 1) / n);
    if (t <= turns && (n == g.tiles_n || n == 8 || live <= AH_L2)) {
      turns = t;
      g.groups = n;
      g.share = share;
    }
  }
  g.error_word = h->error_word;
  if (!sorted && !ah_readable(d_x, ldx)) {  // (the sort copies x anyway)
    ah_align(h->x_own, h->kpad, d_x, ldx, rows, h->in, h->num_sms, st);
    d_x = h->x_own;
    ldx = h->kpad;
  }
  g.x = d_x;
  g.ldx = ldx;
  AhMaps m{h->map_w, h->map_low, {}, h->map_b, h->map_w};
  if (g.share != h->share &&
      !ah_map(&m.low, h->dtype, h->w, h->in, h->out, h->ldw, nvs::AH_BK, (g.share - 1) % nvs::AH_BM + 1,
              CU_TENSOR_MAP_SWIZZLE_128B))
    return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
  if (!ah_map(&m.x, h->dtype, sorted ? h->x_own : d_x, h->in, rows, sorted ? h->kpad : ldx,
              nvs::AH_BK, g.nh, CU_TENSOR_MAP_SWIZZLE_128B) ||
      (g.ids && !ah_map(&m.u, h->dtype, h->u, 256, (int64_t)g.tiles_n * g.max_entries * g.parts * g.block / 16,
                        256, 256, g.per * g.parts * g.bh / 16, CU_TENSOR_MAP_SWIZZLE_NONE)))
    return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
  const bool wide = out_dtype == NCB_DTYPE_F32;
  if (h->dtype == NCB_DTYPE_BF16)
    return ncb_record_status(group == 2 ? ah_head<__nv_bfloat16, 2>(m, g, wide, st)
                                        : ah_head<__nv_bfloat16, 1>(m, g, wide, st));
  return ncb_record_status(group == 2 ? ah_head<__half, 2>(m, g, wide, st)
                                      : ah_head<__half, 1>(m, g, wide, st));
}

}  // extern "C"
