// LM head with low-rank adapters of many requests (sm_100a):
//   out[n, :] = W x_n + scale_s B_s (A_s x_n),  s = adapter_ids[n].
//
// Two kernels. adapter_shrink_kernel computes u_n = scale_s A_s x_n. The batch
// is cut into tiles of NT <= 256 rows; for a tile it lists the slots its rows
// name, 16 ranks of one slot being an entry, and writes each entry's
// [NT, 16] matrix U_e: row n holds u_n where n's adapter is that slot, zeros
// elsewhere. The whole product of a tile is then one sum over a longer inner
// axis,
//   out^T = [W | B_e1 | B_e2 | ...] [x | U_e1 | U_e2 | ...]^T,
// which head_kernel runs on the tensor cores: 128 outputs by NT rows of the
// batch per tile (the weight is the 128-row operand, so that a few rows waste no
// tensor-core rows and every weight byte is read once), accumulated in TMEM. U_e
// is split into two 16-bit values, u = hi + lo, each with its own product: one
// would round u to 8 bits (bf16).
//
// The zeros cost operations, not bytes: reading an entry's B from memory takes
// as long as multiplying it with 256 rows (128 * 16 * 2 bytes against 128 * 16 *
// 2 * 256 * 2 operations per tile).
//
// A weight tile is read once from memory and used for all rows of the batch, so
// up to about 256 rows the head is bound by the weight's bytes, beyond by the
// tensor cores.
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
constexpr int AH_THREADS = 192;   // four epilogue warps, a copying and a multiplying one
constexpr int AH_PAIR = 2;        // adapter entries per stage

struct AhArgs {
  const void* x;
  int64_t ldx;
  int rows, in, kpad, out, slots, slices;  // slices: entries a slot can have
  int nt, tiles_n;                         // rows per tile, tiles of rows
  const int32_t* ids;
  const void* a;        // [slots][16 slices][kpad]
  const int32_t* ranks; // per slot; 0: empty, < 0: |rank|, and B holds a non-finite value
  const float* scales;
  void* u;              // [tiles_n][max_entries][2][nt][16]
  int32_t* entries;     // [tiles_n][max_entries] slot * slices + slice
  int32_t* counts;      // [tiles_n]
  int max_entries;
  void* y;
  int64_t ldo;
  uint32_t idesc;
  int stages;
  uint32_t* error_word;
};

// ---- loading a slot ---------------------------------------------------------------
// B goes to [slice][out][16]: a 128-row tile of an entry is 4 KiB in a row. A
// value of B that is not finite would reach every row of a tile (0 times NaN);
// it is stored as 0 and the slot marked, and the slot's own rows come out as NaN.
template <typename E>
__global__ void adapter_pack_kernel(E* a, E* b, int32_t* ranks, float* scales, int slot, int in,
                                    int kpad, int out, int slices, const E* sa, int64_t lda,
                                    const E* sb, int64_t ldb, int rank) {
  const int64_t na = (int64_t)slices * 16 * kpad, nb = (int64_t)slices * out * 16;
  const int64_t t0 = blockIdx.x * (int64_t)blockDim.x + threadIdx.x, dt = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = t0; i < na; i += dt) {
    const int64_t j = i / kpad, k = i % kpad;
    a[slot * na + i] = j < rank && k < in ? sa[j * lda + k] : E(0.0f);
  }
  bool bad = false;
  for (int64_t i = t0; i < nb; i += dt) {
    const int64_t j = i / ((int64_t)out * 16) * 16 + i % 16, v = i / 16 % out;
    E x = j < rank ? sb[v * ldb + j] : E(0.0f);
    if (!(fabsf((float)x) < INFINITY)) {
      bad = true;
      x = E(0.0f);
    }
    b[slot * nb + i] = x;
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
template <typename E>
__device__ __forceinline__ void ah_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<E, __nv_bfloat16>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int AS_THREADS = 256;

// Eight values of a row of x from column k on; columns past the row are 0.
template <typename E>
__device__ __forceinline__ uint4 ah_row8(const E* row, int k, int in) {
  if (k + 8 <= in) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < in)
      w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[k + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// grid (CTAs, tiles_n). Every CTA lists its tile's entries; the work is dealt out
// as (entry, 16 rows): one 16 x 16 product over the inner axis, eight warps taking
// every eighth 32 columns and their sums added in the order of the warps. It only
// delays the head's last steps, which are the ones that wait for it.
template <typename E>
__global__ void __launch_bounds__(AS_THREADS) adapter_shrink_kernel(const AhArgs g) {
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ uint32_t named[AH_MAX_ADAPTERS / 32];
  __shared__ int32_t ids[AH_NT];
  __shared__ int32_t warp_sum[AS_THREADS / 32];
  __shared__ float part[AS_THREADS / 32][16][17];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, tile = blockIdx.y;
  const int n0 = tile * g.nt;
  int32_t* entries = g.entries + (int64_t)tile * g.max_entries;
  if (t < AH_MAX_ADAPTERS / 32) named[t] = 0;
  __syncthreads();
  if (t < g.nt) {
    int s = n0 + t < g.rows ? g.ids[n0 + t] : -1;
    if (s < 0 || s >= g.slots || g.ranks[s] == 0) s = -1;
    ids[t] = s;
    if (s >= 0) atomicOr(&named[s >> 5], 1u << (s & 31));
  }
  __syncthreads();
  // entries in the order of the slots, four slots per thread
  int mine[4], sum = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int s = 4 * t + j;
    mine[j] = named[s >> 5] >> (s & 31) & 1 ? (abs(g.ranks[s]) + 15) / 16 : 0;
    sum += mine[j];
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int at = inc - sum, count = 0;
#pragma unroll
  for (int w = 0; w < AS_THREADS / 32; ++w) {
    if (w < warp) at += warp_sum[w];
    count += warp_sum[w];
  }
  if (blockIdx.x == 0 && t == 0) g.counts[tile] = count;
  const int blocks = g.nt / 16;
  for (int first = 0; first < count * blocks; first += gridDim.x) {
    const int item = first + blockIdx.x;
    // the thread whose slots hold the item's entry says which it is
    __shared__ int32_t s_slot, s_slice;
    __syncthreads();
    if (item < count * blocks) {
      const int e = item / blocks;
      int b = at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (e >= b && e < b + mine[j]) {
          s_slot = 4 * t + j;
          s_slice = e - b;
        }
        b += mine[j];
      }
    }
    __syncthreads();
    if (item >= count * blocks) continue;
    const int e = item / blocks, r0 = item % blocks * 16;
    const int slot = s_slot, slice = s_slice;
    if (r0 == 0 && t == 0) entries[e] = slot * g.slices + slice;
    const bool any = __syncthreads_or(t < 16 && ids[r0 + t] == slot);
    float u = 0.0f;
    if (any) {
      const E* a = static_cast<const E*>(g.a) +
                   ((int64_t)slot * g.slices + slice) * 16 * (int64_t)g.kpad;
      const int q = lane >> 2, c = (lane & 3) * 8;
      const int na = n0 + r0 + q, nb = na + 8;
      const E* x = static_cast<const E*>(g.x);
      const E* xa = x + (int64_t)min(na, g.rows - 1) * g.ldx;
      const E* xb = x + (int64_t)min(nb, g.rows - 1) * g.ldx;
      const E* pa = a + (int64_t)q * g.kpad;
      const E* pb = a + (int64_t)(q + 8) * g.kpad;
      float acc[2][4] = {};
      // A lane's eight values of a row feed two products: the inner axis may be
      // permuted as long as both operands are.
#pragma unroll 4
      for (int k = warp * 32 + c; k < g.kpad; k += AS_THREADS) {
        const uint4 va = ah_row8(xa, k, g.in), vb = ah_row8(xb, k, g.in);
        const uint4 wa = *reinterpret_cast<const uint4*>(pa + k);
        const uint4 wb = *reinterpret_cast<const uint4*>(pb + k);
        const uint32_t f0[4] = {va.x, vb.x, va.y, vb.y}, f1[4] = {va.z, vb.z, va.w, vb.w};
        ah_mma<E>(acc[0], f0, wa.x, wa.y);
        ah_mma<E>(acc[1], f0, wb.x, wb.y);
        ah_mma<E>(acc[0], f1, wa.z, wa.w);
        ah_mma<E>(acc[1], f1, wb.z, wb.w);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          part[warp][q + 8 * (i >> 1)][8 * h + 2 * (lane & 3) + (i & 1)] = acc[h][i];
      __syncthreads();
      if (ids[r0 + t / 16] == slot) {
        for (int w = 0; w < AS_THREADS / 32; ++w) u += part[w][t / 16][t % 16];
        u *= g.scales[slot];
        if (g.ranks[slot] < 0) u = NAN;
      }
    }
    const E hi = E(u);
    const E lo = E(fabsf((float)hi) < INFINITY ? u - (float)hi : 0.0f);
    E* to = static_cast<E*>(g.u) +
            (((int64_t)tile * g.max_entries + e) * 2 * g.nt + r0) * 16 + t;
    to[0] = hi;
    to[(int64_t)g.nt * 16] = lo;
  }
}

// ---- the product ------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ah_smem(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ bool ah_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// Every wait ends: after about 2 s it gives up.
__device__ __noinline__ bool ah_wait_long(uint32_t bar, uint32_t parity) {
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  do {
    if (ah_try(bar, parity)) return true;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  } while (t - t0 < 2000000000ull);
  return false;
}
__device__ __forceinline__ bool ah_wait(uint32_t bar, uint32_t parity) {
  return ah_try(bar, parity) || ah_try(bar, parity) || ah_wait_long(bar, parity);
}
__device__ __forceinline__ void ah_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void ah_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ah_copy2(uint32_t to, const CUtensorMap* map, uint32_t bar, int x,
                                         int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          to),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void ah_copy3(uint32_t to, const CUtensorMap* map, uint32_t bar, int x,
                                         int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(to),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Shared-memory operand whose rows of `span` bytes (32 or 128) lie one behind the
// other in the TMA's swizzle of that span, eight rows to a group.
__device__ __forceinline__ uint64_t ah_operand(uint32_t addr, int span) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(span * 8 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)(span == 128 ? 2 : 6) << 61;
}
__device__ __forceinline__ void ah_multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc,
                                            bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void ah_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}

template <typename O>
__device__ __forceinline__ O ah_out(uint32_t bits) {
  return O(__uint_as_float(bits));
}

template <typename O>
__global__ void __launch_bounds__(AH_THREADS, 1)
    head_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_u,
                const AhArgs g) {
  extern __shared__ uint8_t ah_raw[];
  __shared__ uint64_t bars[2 * AH_MAX_STAGES + 4];
  __shared__ uint32_t s_tmem;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t stage0 = (ah_smem(ah_raw) + 1023) & ~1023u;
  const uint32_t stage_bytes = AH_A_BYTES + g.nt * 128;
  const uint32_t full = ah_smem(bars), empty = full + 8 * AH_MAX_STAGES,
                 done = empty + 8 * AH_MAX_STAGES, drained = done + 16;
  uint32_t columns = 32;
  while (columns < 2u * g.nt) columns *= 2;
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     ah_smem(&s_tmem)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (t == 0) {
    for (int i = 0; i < AH_MAX_STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8 * i) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty + 8 * i) : "memory");
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(done + 8 * i) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 128;" ::"r"(drained + 8 * i) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const int tiles_m = (g.out + AH_BM - 1) / AH_BM, tiles = tiles_m * g.tiles_n;
  const int steps = (g.in + AH_BK - 1) / AH_BK;

  if (warp == 4) {
    if (lane == 0) {  // ---- copies -----------------------------------------------------
      int s = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true, waited = false;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const int m = tile / g.tiles_n, n = tile % g.tiles_n;
        for (int k = 0; k < steps; ++k) {
          if (!(ok = ah_wait(empty + 8 * s, phase ^ 1))) break;
          const uint32_t a = stage0 + s * stage_bytes, bar = full + 8 * s;
          ah_expect(bar, stage_bytes);
          ah_copy2(a, &map_w, bar, k * AH_BK, m * AH_BM);
          ah_copy2(a + AH_A_BYTES, &map_x, bar, k * AH_BK, n * g.nt);
          ++issued;
          if (++s == g.stages) s = 0, phase ^= 1;
        }
        if (!ok) break;
        if (!waited) {  // what follows reads the shrink kernel's results
          asm volatile("griddepcontrol.wait;" ::: "memory");
          asm volatile("fence.proxy.async.global;" ::: "memory");
          waited = true;
        }
        const int count = g.ids ? *(volatile const int32_t*)(g.counts + n) : 0;
        for (int e = 0; e < count; e += AH_PAIR) {
          if (!(ok = ah_wait(empty + 8 * s, phase ^ 1))) break;
          const int both = count - e < AH_PAIR ? count - e : AH_PAIR;
          const uint32_t a = stage0 + s * stage_bytes, bar = full + 8 * s;
          ah_expect(bar, both * (AH_BM * 32 + 2 * g.nt * 32));
          for (int j = 0; j < both; ++j) {
            ah_copy3(a + j * AH_BM * 32, &map_b, bar, 0, m * AH_BM,
                     *(volatile const int32_t*)(g.entries + (int64_t)n * g.max_entries + e + j));
            const int row = (n * g.max_entries + e + j) * 2 * g.nt;
            ah_copy2(a + AH_A_BYTES + j * g.nt * 64, &map_u, bar, 0, row);
            ah_copy2(a + AH_A_BYTES + j * g.nt * 64 + g.nt * 32, &map_u, bar, 0, row + g.nt);
          }
          ++issued;
          if (++s == g.stages) s = 0, phase ^= 1;
        }
      }
      if (!ok) {  // gave up: no copy may be in flight when the CTA ends
        atomicOr(g.error_word, 1u);
        for (int i = 0; i < g.stages && i < issued; ++i) {
          if (s-- == 0) s = g.stages - 1, phase ^= 1;
          ah_wait(full + 8 * s, phase);
        }
      }
      if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    }
  } else if (warp == 5) {
    if (lane == 0) {  // ---- products -----------------------------------------------------
      int s = 0, turn = 0;
      uint32_t phase = 0;
      bool ok = true, waited = false;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++turn) {
        const int n = tile % g.tiles_n;
        const uint32_t acc = tmem + (turn & 1) * g.nt;
        if (!(ok = ah_wait(drained + 8 * (turn & 1), ((turn >> 1) & 1) ^ 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int k = 0; k < steps; ++k) {
          if (!(ok = ah_wait(full + 8 * s, phase))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t a = ah_operand(stage0 + s * stage_bytes, 128);
          const uint64_t b = ah_operand(stage0 + s * stage_bytes + AH_A_BYTES, 128);
#pragma unroll
          for (int j = 0; j < AH_BK / 16; ++j)
            ah_multiply(acc, a + 2 * j, b + 2 * j, g.idesc, (k | j) != 0);
          ah_commit(empty + 8 * s);
          if (++s == g.stages) s = 0, phase ^= 1;
        }
        if (!ok) break;
        if (!waited) {
          asm volatile("griddepcontrol.wait;" ::: "memory");
          waited = true;
        }
        const int count = g.ids ? *(volatile const int32_t*)(g.counts + n) : 0;
        for (int e = 0; e < count; e += AH_PAIR) {
          if (!(ok = ah_wait(full + 8 * s, phase))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const int both = count - e < AH_PAIR ? count - e : AH_PAIR;
          const uint32_t base = stage0 + s * stage_bytes;
          for (int j = 0; j < both; ++j) {
            const uint64_t a = ah_operand(base + j * AH_BM * 32, 32);
            const uint32_t u = base + AH_A_BYTES + j * g.nt * 64;
            ah_multiply(acc, a, ah_operand(u, 32), g.idesc, true);
            ah_multiply(acc, a, ah_operand(u + g.nt * 32, 32), g.idesc, true);
          }
          ah_commit(empty + 8 * s);
          if (++s == g.stages) s = 0, phase ^= 1;
        }
        if (ok) ah_commit(done + 8 * (turn & 1));
      }
      if (!ok) {
        atomicOr(g.error_word, 2u);
        // products in flight end before TMEM is given back
        ah_commit(done + 8 * (turn & 1));
        ah_wait(done + 8 * (turn & 1), (turn >> 1) & 1);
      }
    }
  } else {  // ---- results ------------------------------------------------------------
    int turn = 0;
    O* y = static_cast<O*>(g.y);
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
      const int m = tile / g.tiles_n, n0 = tile % g.tiles_n * g.nt;
      if (!ah_wait(done + 8 * (turn & 1), (turn >> 1) & 1)) {
        if (t == 0) atomicOr(g.error_word, 4u);
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int v = m * AH_BM + t;  // this lane's output
      const int here = min(g.nt, g.rows - n0);
      const uint32_t acc = tmem + (turn & 1) * g.nt + ((uint32_t)(warp * 32) << 16);
      O* to = y + (int64_t)n0 * g.ldo + v;
      for (int c = 0; c < here; c += 16) {
        uint32_t r[16];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
              "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
              "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(acc + c));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (v < g.out) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < here) to[(int64_t)(c + j) * g.ldo] = ah_out<O>(r[j]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      ah_arrive(drained + 8 * (turn & 1));
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 5)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}

}  // namespace nvs

struct NcbAdapterHead {
  int device = 0, dtype = 0, in = 0, kpad = 0, out = 0, max_rows = 0, slots = 0, max_rank = 0;
  int slices = 0, num_sms = 0;
  std::mutex mu;
  void* mem = nullptr;  // everything below but w and w_own
  void *a = nullptr, *b = nullptr, *u = nullptr, *x_own = nullptr;
  int32_t *ranks = nullptr, *entries = nullptr, *counts = nullptr;
  float* scales = nullptr;
  uint32_t* error_word = nullptr;
  void* w_own = nullptr;  // the weight's copy, where it cannot be read in place
  bool has_w = false;
  CUtensorMap map_w{}, map_b{};
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
// A map of 16-bit values: dims[0] in a row, strides in bytes from dims[1] on.
bool ah_map(CUtensorMap* map, int dtype, const void* base, int rank, const cuuint64_t* dims,
            const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  const cuuint32_t one[3] = {1, 1, 1};
  const AhEncode fn = ah_encode();
  return fn && fn(map, dtype == NCB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool ah_map2(CUtensorMap* map, int dtype, const void* base, int64_t cols, int64_t rows, int64_t ld,
             int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  return ah_map(map, dtype, base, 2, dims, strides, box, swizzle);
}
// Whether a matrix of 16-bit values can be read by tiles in place.
bool ah_readable(const void* p, int64_t ld) { return ah_aligned(p, 16) && ld % 8 == 0; }

template <typename E>
int ah_pack(NcbAdapterHead* h, int slot, const void* a, int64_t lda, const void* b, int64_t ldb,
            int rank, float scale, cudaStream_t st) {
  nvs::adapter_slot_kernel<<<1, 1, 0, st>>>(h->ranks, h->scales, slot, rank, scale);
  nvs::adapter_pack_kernel<E><<<4 * h->num_sms, 256, 0, st>>>(
      static_cast<E*>(h->a), static_cast<E*>(h->b), h->ranks, h->scales, slot, h->in, h->kpad,
      h->out, h->slices, static_cast<const E*>(a), lda, static_cast<const E*>(b), ldb, rank);
  return ah_launched();
}

void ah_align(void* to, int64_t pitch, const void* from, int64_t ld, int64_t rows, int cols,
              int num_sms, cudaStream_t st) {
  const int64_t most = 8LL * num_sms;
  nvs::adapter_align_kernel<uint16_t><<<(unsigned)(rows < most ? rows : most), 256, 0, st>>>(
      static_cast<uint16_t*>(to), pitch, static_cast<const uint16_t*>(from), ld, rows, cols);
}

template <typename O>
int ah_head(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& b, const CUtensorMap& u,
            const nvs::AhArgs& g, int num_sms, cudaStream_t st) {
  const int64_t tiles = (int64_t)((g.out + nvs::AH_BM - 1) / nvs::AH_BM) * g.tiles_n;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles < num_sms ? tiles : num_sms));
  cfg.blockDim = dim3(nvs::AH_THREADS);
  cfg.dynamicSmemBytes = (size_t)g.stages * (nvs::AH_A_BYTES + g.nt * 128) + 1024;
  cfg.stream = st;
  // starts beside the shrink kernel and waits for it where it needs its results
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g.ids ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, nvs::head_kernel<O>, w, x, b, u, g) == cudaSuccess
             ? NCB_OK
             : NCB_ERROR_LAUNCH_FAILED;
}

bool ah_raise() {
  for (const void* fn : {(const void*)nvs::head_kernel<float>, (const void*)nvs::head_kernel<__half>,
                         (const void*)nvs::head_kernel<__nv_bfloat16>})
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
  h->kpad = (in_features + nvs::AH_BK - 1) / nvs::AH_BK * nvs::AH_BK;
  cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device);
  size_t off = 0;
  auto carve = [&](size_t bytes) {
    const size_t o = off;
    off += (bytes + 255) / 256 * 256;
    return o;
  };
  // A batch of n rows is cut into tiles of at most 256, each of a multiple of 16
  // rows, and a tile names at most as many slots as it has rows.
  const size_t tiles = ((size_t)max_rows + nvs::AH_NT - 1) / nvs::AH_NT;
  const size_t most = (size_t)(h->slots < nvs::AH_NT ? h->slots : nvs::AH_NT) * h->slices;
  const size_t rows16 = max_rows > nvs::AH_NT ? (size_t)nvs::AH_NT : ((size_t)max_rows + 15) / 16 * 16;
  const size_t per = (size_t)h->slots * h->slices * 16;
  const size_t o_a = carve(per * h->kpad * 2), o_b = carve(per * h->out * 2);
  const size_t o_x = carve((size_t)max_rows * h->kpad * 2);
  const size_t o_u = carve(tiles * most * 2 * rows16 * 16 * 2);
  const size_t o_e = carve(tiles * most * 4), o_c = carve(tiles * 4);
  const size_t o_s = carve((size_t)h->slots * 4), o_r = carve((size_t)h->slots * 4);
  const size_t o_w = carve(4);
  if (cudaMalloc(&h->mem, off) != cudaSuccess) {
    cudaGetLastError();
    delete h;
    return ncb_record_status(NCB_ERROR_ALLOC_FAILED);
  }
  char* m = static_cast<char*>(h->mem);
  h->a = m + o_a;
  h->b = m + o_b;
  h->x_own = m + o_x;
  h->u = m + o_u;
  h->entries = reinterpret_cast<int32_t*>(m + o_e);
  h->counts = reinterpret_cast<int32_t*>(m + o_c);
  h->scales = reinterpret_cast<float*>(m + o_s);
  h->ranks = reinterpret_cast<int32_t*>(m + o_r);
  h->error_word = reinterpret_cast<uint32_t*>(m + o_w);
  bool ok = ah_raise() && cudaMemset(h->ranks, 0, off - o_r) == cudaSuccess &&
            cudaDeviceSynchronize() == cudaSuccess;
  if (ok && h->slots) {  // [slot and slice][out][16]
    const cuuint64_t dims[3] = {16, (cuuint64_t)h->out, (cuuint64_t)h->slots * h->slices};
    const cuuint64_t strides[2] = {32, (cuuint64_t)h->out * 32};
    const cuuint32_t box[3] = {16, nvs::AH_BM, 1};
    ok = ah_map(&h->map_b, dtype, h->b, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_32B);
  }
  if (!ok) {
    cudaGetLastError();
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
    cudaFree(h->w_own);
  }
  delete h;
  return ncb_record_status(NCB_OK);
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
  h->has_w = ah_map2(&h->map_w, h->dtype, d_weight, h->in, h->out, ld, nvs::AH_BK, nvs::AH_BM,
                     CU_TENSOR_MAP_SWIZZLE_128B);
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
  std::lock_guard<std::mutex> lk(h->mu);
  AhDevice guard(h->device);
  if (!guard.ok) return ncb_record_status(NCB_ERROR_INIT_FAILED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!ah_readable(d_x, ldx)) {
    ah_align(h->x_own, h->kpad, d_x, ldx, rows, h->in, h->num_sms, st);
    d_x = h->x_own;
    ldx = h->kpad;
  }
  nvs::AhArgs g{};
  g.x = d_x;
  g.ldx = ldx;
  g.rows = rows;
  g.in = h->in;
  g.kpad = h->kpad;
  g.out = h->out;
  g.slots = h->slots;
  g.slices = h->slices;
  g.tiles_n = (rows + nvs::AH_NT - 1) / nvs::AH_NT;
  g.nt = ((rows + g.tiles_n - 1) / g.tiles_n + 15) / 16 * 16;
  g.ids = h->slots ? d_adapter_ids : nullptr;
  g.a = h->a;
  g.ranks = h->ranks;
  g.scales = h->scales;
  g.u = h->u;
  g.entries = h->entries;
  g.counts = h->counts;
  g.max_entries = (h->slots < g.nt ? h->slots : g.nt) * h->slices;
  g.y = d_out;
  g.ldo = ldo;
  const uint32_t type = h->dtype == NCB_DTYPE_BF16 ? 1u : 0u;
  // fp32 sums, both operands of the head's type with the inner axis in rows
  g.idesc = 1u << 4 | type << 7 | type << 10 | (uint32_t)(g.nt / 8) << 17 | (nvs::AH_BM / 16) << 24;
  const int stage = nvs::AH_A_BYTES + g.nt * 128;
  g.stages = nvs::AH_SMEM / stage < nvs::AH_MAX_STAGES ? nvs::AH_SMEM / stage : nvs::AH_MAX_STAGES;
  g.error_word = h->error_word;
  CUtensorMap map_x, map_u = h->map_w;
  if (!ah_map2(&map_x, h->dtype, d_x, h->in, rows, ldx, nvs::AH_BK, g.nt, CU_TENSOR_MAP_SWIZZLE_128B) ||
      (g.ids && !ah_map2(&map_u, h->dtype, h->u, 16, (int64_t)g.tiles_n * g.max_entries * 2 * g.nt, 16,
                         16, g.nt, CU_TENSOR_MAP_SWIZZLE_32B)))
    return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
  if (g.ids) {
    const int64_t items = (int64_t)g.max_entries * (g.nt / 16);
    const int per_tile = (h->num_sms + g.tiles_n - 1) / g.tiles_n;
    const dim3 grid((unsigned)(items < per_tile ? items : per_tile), g.tiles_n);
    if (h->dtype == NCB_DTYPE_BF16)
      nvs::adapter_shrink_kernel<__nv_bfloat16><<<grid, nvs::AS_THREADS, 0, st>>>(g);
    else
      nvs::adapter_shrink_kernel<__half><<<grid, nvs::AS_THREADS, 0, st>>>(g);
    if (ah_launched() != NCB_OK) return ncb_record_status(NCB_ERROR_LAUNCH_FAILED);
  }
  return ncb_record_status(out_dtype == NCB_DTYPE_F32
                               ? ah_head<float>(h->map_w, map_x, h->map_b, map_u, g, h->num_sms, st)
                           : h->dtype == NCB_DTYPE_BF16
                               ? ah_head<__nv_bfloat16>(h->map_w, map_x, h->map_b, map_u, g, h->num_sms, st)
                               : ah_head<__half>(h->map_w, map_x, h->map_b, map_u, g, h->num_sms, st));
}

}  // extern "C"
