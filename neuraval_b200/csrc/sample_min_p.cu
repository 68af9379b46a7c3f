// Sampling with options per row, min-p and 16-bit logits (sm_100a).
//
//   order: x descending, id ascending;  w_i = exp((x_i - max) / T)
//   K = the first top_k of the order, of mass Z;  P = the shortest prefix of K of
//   mass >= top_p Z;  M = {w_i >= min_p} in P;  token = the first of the order
//   whose prefix mass exceeds u mass(M).
//
// Every set is a prefix of the order, so a row needs no sort, only the places
// where a count (top_k), a value (min_p) or a mass (top_p, the draw) is crossed.
// Rows of 16-bit values have a kernel of their own, further down, which counts each
// value; this is the one for fp32 rows. A row belongs to a cluster of 1..8 CTAs (more
// CTAs for few rows). CTA 0 decides, the others carry out its commands:
//   1. few values wanted (the usual options): each thread's maximum of the first
//      quarter or half of the row; the k-th largest of them is a lower bound of the
//      k-th value, min-p has one of its own. The rest is read once, what is above the
//      bound listed (each CTA its own, then one list), sorted by (x, id), and
//      everything is decided on 64-bit prefix sums of the list. The row crosses HBM
//      once: 256x128256 takes 65 us, 2.0 TB/s, its floor being 20; what is left
//      is the list's sort and the cluster's and the block's barriers, of which two
//      CTAs to an SM hide a part.
//   2. Otherwise the maximum and the least finite value (NaN and +inf show in a
//      NaN-propagating maximum) of all of it; the passes that follow mostly read L2.
//   3. Otherwise, or where the list overflows: a histogram of counts over SP_BINS
//      equal steps of x below the maximum (integers: their order does not matter).
//      It gives the bin of the k-th value exactly, and about where the masses are
//      crossed. One more pass sums the exact 64-bit weights above each guessed
//      window of bins and gathers the windows; a crossing outside its window moves
//      the window and repeats the pass; a window with more values than a list holds
//      is one value many times, whose crossing is a division, or is divided by a
//      histogram of the values' bits.
// Sums run in an order fixed by the sizes alone; the lists' order of arrival is
// sorted away.
//
// Keeping a cluster's slices of the row in shared memory, for one read in all, was
// slower: it leaves two CTAs per SM in long chains of small steps, and more of them
// per row to synchronise (1024x151936 with top-p alone: 2.3 ms, now 0.95, of which
// the 64-bit weights of the exact pass are the largest part: it issues about 30
// operations per value). A crossing in a bin of more than SP_CAP values takes up to seven
// passes: one row in a hundred of 256x128256 with top-p alone, peaked at few values,
// which then decide how long the call takes (1.4 ms).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "navsampler.h"
#include "sample_search.cuh"

int ncb_record_status(int st);

namespace nvs {
namespace cg = cooperative_groups;

constexpr int SP_NT = 512;       // threads of a CTA
constexpr int SP_BINS = 2048;    // histogram bins (four per thread)
constexpr int SP_FEW = 1024;     // values that one list holds and sorts
constexpr int SP_CAP = 512;      // and one window's part of the list
constexpr int SP_WIDEN = 96;     // values up to which a guessed window takes in its neighbours
constexpr int SP_RANKED = 256;   // lists up to this are sorted by ranks
constexpr int SP_SOME = 512;     // bins of which a value is kept, for the guess
// Largest top_k that the threads' maxima bound: half of a CTA's threads (with hardly more
// maxima than values wanted the bound is so low that the list overflows). 256x128256 fp32, all rows alike: top_k 50 55 us, 256 72; from
// 257 on the histogram decides, 110 us, 121 for 1000.
constexpr int SP_BOUNDED = 256;
constexpr int SP_CLUSTER = 8;    // largest cluster
constexpr int SP_TURNS = 4096;   // passes over a row at most
constexpr int SP_MAX_VOCAB = 1 << 24;
// Values further than this below the maximum (in units of T) carry no mass:
// 2^24 of them weigh less than 2^24 e^-60 = 1.5e-19 of the maximum's own weight,
// below the 2^-53 at which 64-bit sums round.
constexpr double SP_REACH = 60.0;

struct SpArgs {
  const void* logits;
  int64_t ld;
  int vocab;
  int per;  // 16-byte granules per CTA
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  float* logprobs;
  int32_t* kept;
  uint32_t* flags;
};

enum { SP_DONE, SP_FIRST, SP_PASS, SP_HIST, SP_GATHER, SP_STREAM, SP_SELECT };
enum { SP_K = 0, SP_P = 1, SP_D = 2, SP_WINDOWS = 3 };

struct SpCmd {
  int op;
  float high[SP_WINDOWS], low[SP_WINDOWS];  // SP_FIRST: each window's values, both ends in it
  uint32_t klo[SP_WINDOWS], khi[SP_WINDOWS];  // each window's keys, both ends in it
  int gather[SP_WINDOWS];                     // whether its values are listed
  float theta;                                // least value that min-p keeps; SP_GATHER: least wanted
  int shift;                                  // SP_HIST: bin = (khi[0] - key) >> shift; < 0: bin(value)
  float value;                                // SP_SELECT: the value and which of its
  int nth;                                    //   occurrences, by id
};

// What a pass adds up: mass and count above each window, then at or above theta,
// then in each window.
constexpr int SP_SUMS = 2 * SP_WINDOWS + 1;
struct SpPart {
  double mass[SP_SUMS];
  int n[SP_SUMS];
  __device__ __forceinline__ double above(int w) const { return mass[w]; }
  __device__ __forceinline__ double in(int w) const { return mass[SP_WINDOWS + 1 + w]; }
  __device__ __forceinline__ int n_above(int w) const { return n[w]; }
  __device__ __forceinline__ int n_in(int w) const { return n[SP_WINDOWS + 1 + w]; }
};

struct SpShared {
  uint4 hist4[SP_BINS / 4];  // counts; in CTA 0, once merged, the counts before each bin
  uint4 some4[SP_SOME / 4];  // a value of each filled bin, of the first bins (sp_ticket)
  alignas(16) float mass[SP_BINS + 4];  // CTA 0, once merged: about the mass before each bin
  unsigned long long list[SP_WINDOWS * SP_CAP];
  SpCmd cmd;
  SpPart part[SP_CLUSTER];
  float mx[SP_CLUSTER], mn[SP_CLUSTER];
  int count[SP_CLUSTER];
  int n_list[SP_WINDOWS];
  uint32_t k_low[SP_CLUSTER][SP_WINDOWS], k_high[SP_CLUSTER][SP_WINDOWS];  // least and greatest key in a window
  int token;
  int total;  // finite values of the row
  // scratch of the block-wide steps
  double red_d[SP_NT / 32];
  float red_f[SP_NT / 32];
  int red_i[SP_NT / 32];
  SpPart warp_part[SP_NT / 32];
  double got_d;
  int got_i, bin_k, bin_last;
  float theta;
  uint32_t tops[2 * SP_WINDOWS];
};

// The CTA's shared memory, by a name that is known to be shared: through a pointer in
// SpRow every access would be a generic one.
extern __shared__ uint4 sp_raw[];
__device__ __forceinline__ SpShared& sp_shared() { return *reinterpret_cast<SpShared*>(sp_raw); }

// A bin's stand-in is the value with the greatest ticket: as good as any of them, but not
// one that depends on timing, since the order of the sums follows from what is guessed by
// it. (The greatest value itself made the guesses too high: 5 us of 1024x151936 flat.)
__device__ __forceinline__ uint32_t sp_ticket(float v) { return __brev(__float_as_uint(v)); }
__device__ __forceinline__ float sp_drawn(uint32_t ticket) { return __uint_as_float(__brev(ticket)); }
// A window's greatest key as a value. (No value has the key of -0; as a float it would
// take +0 with it.)
__device__ __forceinline__ float sp_edge(uint32_t k) {
  return sp_value(k == 0x7FFFFFFFu ? 0x7FFFFFFEu : k);
}
__device__ __forceinline__ float sp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename E>
struct SpVec;
template <>
struct SpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& g, float* v) {
    v[0] = __uint_as_float(g.x);
    v[1] = __uint_as_float(g.y);
    v[2] = __uint_as_float(g.z);
    v[3] = __uint_as_float(g.w);
  }
  static __device__ __forceinline__ uint32_t none() { return 0xFF800000u; }
};
template <>
struct SpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& g, float* v) {
    const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint32_t none() { return 0xFF80u; }
};
template <>
struct SpVec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& g, float* v) {
    const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint32_t none() { return 0xFC00u; }
};

// The row passes by the L1 cache: what does not fit into registers lives there.
__device__ __forceinline__ uint4 sp_load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// A CTA's slice: 16-byte granules [g0, g0 + n) of the row, granule 0 starting at
// the 16-byte boundary at or below the row's first value. Only the row's first and
// last granule can hold values of other rows; they are read value by value and
// filled up with -inf.
template <typename E>
struct SpSlice {
  const char* base;  // the row's first granule
  int skip;          // values of granule 0 before the row's first
  int vocab, g0, n;

  // Granule i of the slice, whole or not.
  __device__ __noinline__ uint4 fetch(int i) const {
    constexpr int N = SpVec<E>::N;
    const int g = g0 + i, first = g * N - skip;
    if (first >= 0 && first + N <= vocab) return __ldg(reinterpret_cast<const uint4*>(base) + g);
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (sizeof(E) == 4) {
        const int id = first + q;
        w[q] = id >= 0 && id < vocab
                   ? *reinterpret_cast<const uint32_t*>(base + 16 * (int64_t)g + 4 * q)
                   : SpVec<E>::none();
      } else {
        w[q] = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int id = first + 2 * q + h;
          const uint32_t x =
              id >= 0 && id < vocab
                  ? *reinterpret_cast<const uint16_t*>(base + 16 * (int64_t)g + 4 * q + 2 * h)
                  : SpVec<E>::none();
          w[q] |= x << (16 * h);
        }
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // f(values, granule) for this thread's granules, FLIGHT loads at a time. The whole
  // granules are read without a branch (the loads would wait for one another); past
  // the end the last one is read again and dropped.
  // Granules [begin, end) of the slice.
  template <int FLIGHT, int THREADS, typename F>
  __device__ __forceinline__ void each_granule(F f, int begin, int end) const {
    constexpr int N = SpVec<E>::N;
    const bool front = begin == 0 && end > 0 && g0 * N < skip,
               back = end == n && end > begin + (front ? 1 : 0) && (g0 + n) * N - skip > vocab;
    const int lo = begin + (front ? 1 : 0), hi = end - (back ? 1 : 0);
    const uint4* from = reinterpret_cast<const uint4*>(base) + g0;
    uint4 g[FLIGHT];
    auto load = [&](int i0) {
#pragma unroll
      for (int j = 0; j < FLIGHT; ++j) g[j] = sp_load(from + min(i0 + j * THREADS, hi - 1));
    };
    const int i0 = lo + threadIdx.x;
    if constexpr (FLIGHT < 4) {
      if (lo < hi) load(i0);
#pragma unroll 1
      for (int i = i0; i < hi; i += FLIGHT * THREADS) {
        uint4 now[FLIGHT];
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j) now[j] = g[j];
        load(i + FLIGHT * THREADS);  // on its way while f works
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j)
          if (i + j * THREADS < hi) f(now[j], i + j * THREADS);
      }
    } else {  // light work: the other warps' loads are on their way
#pragma unroll 1
      for (int i = i0; i < hi; i += FLIGHT * THREADS) {
        load(i);
#pragma unroll
        for (int j = 0; j < FLIGHT; ++j)
          if (i + j * THREADS < hi) f(g[j], i + j * THREADS);
      }
    }
    const int edge = threadIdx.x == 0 && front ? 0 : threadIdx.x == 32 && back ? n - 1 : -1;
    if (edge >= 0) f(fetch(edge), edge);
  }
  template <int FLIGHT, typename F>
  __device__ __forceinline__ void each(F f, int begin, int end) const {
    each_granule<FLIGHT, SP_NT>([&](const uint4& g, int i) {
      float v[SpVec<E>::N];
      SpVec<E>::get(g, v);
      f(v, i);
    }, begin, end);
  }
  template <int FLIGHT, typename F>
  __device__ __forceinline__ void each(F f) const {
    each<FLIGHT>(f, 0, n);
  }
  // Of the row at x, the part of CTA `rank`: `per` granules.
  __device__ __forceinline__ void set(const E* x, int vocab_, int rank, int per) {
    constexpr int N = SpVec<E>::N;
    skip = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(E));
    base = reinterpret_cast<const char*>(x - skip);
    vocab = vocab_;
    const int granules = (vocab + skip + N - 1) / N;
    g0 = min(granules, rank * per);
    n = min(granules, (rank + 1) * per) - g0;
  }
  __device__ __forceinline__ int id(int i, int e) const {
    return (g0 + i) * SpVec<E>::N - skip + e;
  }
};

// exp(d c ln2) for 0 >= d c > -1000: with d c = n + r, n whole, |r| <= 1/2, it is 2^n
// times the series of exp(r ln2), cut off after r^11 (6e-15 of it). Own code, for the
// range that is needed: a pass over a row is bound by these operations. (A table of
// 1024 values and three terms took as long: random reads of shared memory.)
__device__ __forceinline__ double sp_exp(double d, double c) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: rounds to a whole number
  constexpr double l = 0.69314718055994530942, l2 = l * l, l4 = l2 * l2, l8 = l4 * l4;
  const double t = fma(d, c, magic);
  const double r = fma(d, c, magic - t), r2 = r * r, r4 = r2 * r2;
  const double a = fma(r, l, 1.0), b = fma(r, l2 * l / 6.0, l2 / 2.0),
               e = fma(r, l4 * l / 120.0, l4 / 24.0), f = fma(r, l4 * l2 * l / 5040.0, l4 * l2 / 720.0),
               g = fma(r, l8 * l / 362880.0, l8 / 40320.0),
               h = fma(r, l8 * l2 * l / 39916800.0, l8 * l2 / 3628800.0);
  const double w = fma(fma(fma(h, r2, g), r4, fma(f, r2, e)), r4, fma(b, r2, a));
  return __hiloint2double(__double2hiint(w) + (__double2loint(t) << 20), __double2loint(w));
}

template <typename T>
__device__ __forceinline__ T sp_warp_scan(T v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T x = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += x;
  }
  return v;
}
// Exclusive prefix over the block's threads, in thread order; `total` to all.
template <typename T>
__device__ __forceinline__ T sp_block_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T inc = sp_warp_scan(v);
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SP_NT / 32; ++i) {
    if (i < warp) before += red[i];
    all += red[i];
  }
  __syncthreads();
  *total = all;
  return before + (inc - v);
}
__device__ __forceinline__ int sp_block_sum(int v, int* red) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < SP_NT / 32; ++i) all += red[i];
  __syncthreads();
  return all;
}

// Sorts a list, largest first. Short ones by their ranks: several threads count the
// larger entries for each. Longer ones bitonically; places [n, power of two) are
// filled with 0, which no listed value has (its low half is never 0).
__device__ __noinline__ void sp_sort(unsigned long long* list, int n) {
  if (n <= SP_RANKED) {
    const int log = n <= 64 ? 3 : n <= 128 ? 2 : 1, per = 1 << log;  // threads per entry
    const int i = threadIdx.x >> log, part = threadIdx.x & (per - 1);
    unsigned long long mine = 0;
    int rank = 0;
    if (i < n) {
      mine = list[i];
      for (int j = part; j < n; j += per) rank += list[j] > mine;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
      if (o < per) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    __syncthreads();
    if (i < n && part == 0) list[rank] = mine;
    __syncthreads();
    return;
  }
  int p = 2 * SP_RANKED;
  while (p < n) p <<= 1;
  for (int i = n + threadIdx.x; i < p; i += SP_NT) list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= p; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < p / 2; i += SP_NT) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const bool down = (lo & size) == 0;
        const unsigned long long x = list[lo], y = list[hi];
        if ((x < y) == down) {
          list[lo] = y;
          list[hi] = x;
        }
      }
      __syncthreads();
    }
}

__device__ void sp_write(const SpArgs& a, int row, int token, float logprob, int kept,
                         uint32_t flags) {
  a.tokens[row] = token;
  if (a.logprobs) a.logprobs[row] = logprob;
  if (a.kept) a.kept[row] = kept;
  if (a.flags) a.flags[row] = flags;
}

__device__ void sp_write_bad(const SpArgs& a, int row, uint32_t flag) {
  sp_write(a, row, -1, __uint_as_float(0x7FC00000u), 0, flag);
}

struct SpOptions {
  float T, top_p, min_p, u;
  int top_k;
  __device__ __forceinline__ bool read(const SpArgs& a, int row) {
    T = a.temperature ? a.temperature[row] : 1.0f;
    top_k = a.top_k ? a.top_k[row] : 0;
    top_p = a.top_p ? a.top_p[row] : 1.0f;
    min_p = a.min_p ? a.min_p[row] : 0.0f;
    u = a.uniforms[row];
    return T >= 0.0f && T <= FLT_MAX &&
           (T == 0.0f || (top_p > 0.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f));
  }
};

__device__ float sp_least_kept(float mx, float T, float min_p, double inv_t) {
  return sp_least_kept(mx, T, min_p, inv_t, [] {});
}

// What a value of the row means. The passes work on a copy of their own: behind a
// pointer, every store to shared memory would have it read again.
struct SpView {
  float mx;           // the row's maximum
  double c;           // 1 / (T ln 2)
  double inv_t;
  float scale;        // bins per unit of x
  float zero;         // values below carry no mass (SP_REACH)

  // A value's place among the bins; its whole part is the bin, the last bin has all
  // further places.
  __device__ __forceinline__ float place(float v) const {  // (finite: what is below INFINITY)
    return fminf((mx - v) * scale, FLT_MAX);
  }
  __device__ __forceinline__ int bin(float v) const {
    return min(SP_BINS - 1, __float2int_rd(place(v)));
  }
  __device__ __forceinline__ double weight(float v) const {
    return sp_exp((double)v - (double)mx, c);
  }
  // of a listed value
  __device__ __forceinline__ double weight_any(float v) const {
    return exp(((double)v - (double)mx) * inv_t);
  }
};

template <typename E>
struct SpRow {
  SpSlice<E> sl;
  cg::cluster_group cl;
  int rank, ranks;
  float T;
  int part;  // granules of the slice that the first pass looks at
  SpView k;

  // Greatest and least finite value of the CTA's threads to every CTA of the row.
  __device__ void share(float mx, float mn) {
    SpShared& s = sp_shared();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = sp_max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if ((threadIdx.x & 31) == 0) {
      s.red_f[threadIdx.x >> 5] = mx;
      s.red_i[threadIdx.x >> 5] = __float_as_int(mn);
    }
    __syncthreads();
    if (threadIdx.x < ranks) {
      for (int w = 0; w < SP_NT / 32; ++w) {
        mx = sp_max_nan(mx, s.red_f[w]);
        mn = fminf(mn, __int_as_float(s.red_i[w]));
      }
      of(threadIdx.x).mx[rank] = mx;
      of(threadIdx.x).mn[rank] = mn;
    }
  }
  // From what all have shared: the maximum, and what values mean below it.
  __device__ float view() {
    SpShared& s = sp_shared();
    float mx = s.mx[0], mn = s.mn[0];
    for (int r = 1; r < ranks; ++r) {
      mx = sp_max_nan(mx, s.mx[r]);
      mn = fminf(mn, s.mn[r]);
    }
    k.mx = mx;
    k.inv_t = 1.0 / (double)T;
    k.c = k.inv_t / 0.69314718055994530942;
    // bins over the finite values, as far as they carry mass
    const double far = (double)mx - SP_REACH * (double)T;
    k.zero = far > -(double)FLT_MAX ? (float)far : -FLT_MAX;
    k.scale = (float)fmin((SP_BINS - 1) / ((double)mx - fmax((double)mn, far)), (double)FLT_MAX);
    return mx;
  }
  static __device__ __forceinline__ bool finite(float x) { return x >= -FLT_MAX && x <= FLT_MAX; }
  template <bool LIST>
  static __device__ __forceinline__ void take(const SpSlice<E>& sl, const float* v, int i, float least,
                                              float& mx, float& mn) {
    float most = v[0];
#pragma unroll
    for (int e = 0; e < SpVec<E>::N; ++e) {
      if (e) most = sp_max_nan(most, v[e]);
      mn = fminf(mn, v[e] == -INFINITY ? INFINITY : v[e]);
    }
    mx = sp_max_nan(mx, most);
    if (LIST && !(most < least)) {  // (or a NaN, which hides the others; the row is bad then)
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e)
        if (v[e] >= least) put(0, 0, SP_FEW, v[e], sl.id(i, e));
    }
  }

  __device__ __forceinline__ SpShared& of(int r) { return *cl.map_shared_rank(&sp_shared(), r); }

  // ---- the commands, carried out by every CTA of the cluster ------------------
  __device__ __noinline__ void hist_by_value() {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    const SpView k = this->k;
    sl.template each<2>([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e)
        if (v[e] > -INFINITY) {
          const int b = k.bin(v[e]);
          atomicAdd(reinterpret_cast<int*>(s.hist4) + b, 1);
          if (b < SP_SOME) atomicMax(reinterpret_cast<uint32_t*>(s.some4) + b, sp_ticket(v[e]));
        }
    });
  }
  __device__ __noinline__ void hist_by_key(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    sl.template each<1>([&](const float* v, int) {
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e) {
        const uint32_t k = sp_key(v[e]);
        if (k >= m.klo[0] && k <= m.khi[0]) {
          const uint32_t b = (m.khi[0] - k) >> m.shift;
          atomicAdd(reinterpret_cast<int*>(s.hist4) + b, 1);
        }
      }
    });
  }
  // A value into the CTA's own list w (places [base, base + cap) of `list`). CTA 0's is
  // the row's; the others hand theirs over after a pass (an atomic on another CTA's
  // memory holds a warp up for a microsecond; a call that is not inlined, three).
  static __device__ __forceinline__ void put(int w, int base, int cap, float v, int id) {
    SpShared& s = sp_shared();
    const int at = atomicAdd(&s.n_list[w], 1);
    if (at < cap)
      s.list[base + at] = ((unsigned long long)sp_key(v) << 32) | (0xFFFFFFFFu - (uint32_t)id);
  }
  __device__ void hand_over(int w, int base, int cap) {
    if (rank == 0) return;
    SpShared& s = sp_shared();
    SpShared& to = of(0);
    __syncthreads();
    const int n = s.n_list[w];
    if (n == 0) return;
    if (threadIdx.x == 0) s.got_i = atomicAdd(&to.n_list[w], n);
    __syncthreads();
    const int at = s.got_i;
    for (int i = threadIdx.x; i < min(n, cap); i += SP_NT)
      if (at + i < cap) to.list[base + at + i] = s.list[base + i];
    __syncthreads();
    if (threadIdx.x == 0) s.n_list[w] = 0;
  }
  __device__ __noinline__ void gather(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    const float least = m.theta;
    float mx = -INFINITY, mn = INFINITY;
    sl.template each<4>([&](const float* v, int i) { take<true>(sl, v, i, least, mx, mn); });
    hand_over(0, 0, SP_FEW);
  }
  // What the first pass left, with its maximum, and the values from `theta` on of all.
  __device__ __noinline__ void stream(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    const float least = m.theta;
    float mx = s.mx[rank], mn = s.mn[rank];
    sl.template each<4>([&](const float* v, int i) { take<true>(sl, v, i, least, mx, mn); }, part, sl.n);
    sl.template each<4>([&](const float* v, int i) { take<true>(sl, v, i, least, mx, mn); }, 0, part);
    hand_over(0, 0, SP_FEW);
    __syncthreads();
    share(mx, mn);
  }
  // The usual pass: windows that are runs of bins. Exact masses above each and of what
  // min-p keeps; the values of a window into its list, or, where they are too many,
  // their least and greatest key (they may all be one value).
  // WITH_K: K's mass ends at a window too (otherwise it is the row's); WITH_M: min-p is on.
  template <bool WITH_K, bool WITH_M>
  __device__ __noinline__ void first_pass(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    const SpView k = this->k;
    SpShared& to = of(0);
    float lo[SP_WINDOWS], hi[SP_WINDOWS];
#pragma unroll
    for (int w = 0; w < SP_WINDOWS; ++w) {
      lo[w] = m.low[w];
      hi[w] = m.high[w];
    }
    const float theta = m.theta;
    double mass[SP_WINDOWS + 1] = {};
    uint32_t low[SP_WINDOWS], high[SP_WINDOWS];
#pragma unroll
    for (int w = 0; w < SP_WINDOWS; ++w) low[w] = 0xFFFFFFFFu, high[w] = 0;
    int n = 0;
    sl.template each<1>([&](const float* v, int i) {
      uint32_t in = 0;  // values of the granule in some window
#pragma unroll
      for (int e0 = 0; e0 < SpVec<E>::N; e0 += 2) {
        double wt[2];  // two at a time: each is a long chain of 64-bit operations
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // out of reach: weighed as if just within it, and not added
          const float x = v[e0 + h];
          wt[h] = k.weight(fmaxf(x, k.zero));
          if (!(x >= k.zero)) wt[h] = 0.0;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = v[e0 + h];
          bool at = false;
#pragma unroll
          for (int w = WITH_K ? SP_K : SP_P; w < SP_WINDOWS; ++w) {
            if (x > hi[w]) mass[w] += wt[h];
            at |= x <= hi[w] && x >= lo[w];
          }
          if (!WITH_K) mass[SP_K] += wt[h];
          if (at) in |= 1u << (e0 + h);
          if (WITH_M && x >= theta) {
            mass[SP_WINDOWS] += wt[h];
            ++n;
          }
        }
      }
      if (in) {
#pragma unroll
        for (int e = 0; e < SpVec<E>::N; ++e) {
          if (!(in >> e & 1)) continue;
          const float x = v[e];
#pragma unroll
          for (int w = 0; w < SP_WINDOWS; ++w)
            if (x <= hi[w] && x >= lo[w]) {
              if (m.gather[w]) {
                put(w, w * SP_CAP, SP_CAP, x, sl.id(i, e));
              } else {
                low[w] = min(low[w], sp_key(x));
                high[w] = max(high[w], sp_key(x));
              }
            }
        }
      }
    });
    for (int w = 0; w < SP_WINDOWS; ++w)
      if (m.gather[w]) hand_over(w, w * SP_CAP, SP_CAP);
#pragma unroll
    for (int j = 0; j <= SP_WINDOWS; ++j)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mass[j] += __shfl_xor_sync(0xffffffffu, mass[j], o);
    n = __reduce_add_sync(0xffffffffu, n);
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int w = 0; w < SP_WINDOWS; ++w) {
      low[w] = __reduce_min_sync(0xffffffffu, low[w]);
      high[w] = __reduce_max_sync(0xffffffffu, high[w]);
    }
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int j = 0; j <= SP_WINDOWS; ++j) s.warp_part[warp].mass[j] = mass[j];
      s.warp_part[warp].n[SP_WINDOWS] = n;
#pragma unroll
      for (int w = 0; w < SP_WINDOWS; ++w) {
        s.warp_part[warp].n[w] = (int)low[w];
        s.warp_part[warp].n[SP_WINDOWS + 1 + w] = (int)high[w];
      }
    }
    __syncthreads();
    const int j = threadIdx.x & 31;
    if (threadIdx.x <= SP_WINDOWS) {
      double sum = 0.0;
      for (int w = 0; w < SP_NT / 32; ++w) sum += s.warp_part[w].mass[j];
      to.part[rank].mass[j] = sum;
    } else if (warp == 1 && j < SP_SUMS) {
      int sum = 0;
      uint32_t least = 0xFFFFFFFFu, most = 0;
      for (int w = 0; w < SP_NT / 32; ++w) {
        const int x = s.warp_part[w].n[j];
        sum += x;
        least = min(least, (uint32_t)x);
        most = max(most, (uint32_t)x);
      }
      if (j < SP_WINDOWS) to.k_low[rank][j] = least;
      else if (j == SP_WINDOWS) to.part[rank].n[j] = sum;
      else to.k_high[rank][j - SP_WINDOWS - 1] = most;
    }
    __syncthreads();
  }
  // Any windows, by their keys, with what lies in them; those that fit are listed.
  __device__ __noinline__ void pass(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    const SpView k = this->k;
    SpShared& to = of(0);
    float lo[SP_WINDOWS], hi[SP_WINDOWS];
#pragma unroll
    for (int w = 0; w < SP_WINDOWS; ++w) {
      lo[w] = sp_value(m.klo[w]);
      hi[w] = sp_edge(m.khi[w]);
    }
    SpPart p{};
    sl.template each<1>([&](const float* v, int i) {
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e) {
        const float x = v[e];
        if (!(x > -INFINITY)) continue;
        const double wt = x >= k.zero ? k.weight(x) : 0.0;
#pragma unroll
        for (int w = 0; w < SP_WINDOWS; ++w) {
          if (x > hi[w]) {
            p.mass[w] += wt;
            ++p.n[w];
          } else if (x >= lo[w]) {
            p.mass[SP_WINDOWS + 1 + w] += wt;
            ++p.n[SP_WINDOWS + 1 + w];
            if (m.gather[w]) put(w, w * SP_CAP, SP_CAP, x, sl.id(i, e));
          }
        }
        if (x >= m.theta) {
          p.mass[SP_WINDOWS] += wt;
          ++p.n[SP_WINDOWS];
        }
      }
    });
    for (int w = 0; w < SP_WINDOWS; ++w)
      if (m.gather[w]) hand_over(w, w * SP_CAP, SP_CAP);
#pragma unroll
    for (int j = 0; j < SP_SUMS; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) p.mass[j] += __shfl_xor_sync(0xffffffffu, p.mass[j], o);
      p.n[j] = __reduce_add_sync(0xffffffffu, p.n[j]);
    }
    if ((threadIdx.x & 31) == 0) s.warp_part[threadIdx.x >> 5] = p;
    __syncthreads();
    if (threadIdx.x < SP_SUMS) {
      double mass = 0.0;
      int n = 0;
      for (int w = 0; w < SP_NT / 32; ++w) {
        mass += s.warp_part[w].mass[threadIdx.x];
        n += s.warp_part[w].n[threadIdx.x];
      }
      to.part[rank].mass[threadIdx.x] = mass;
      to.part[rank].n[threadIdx.x] = n;
    }
    __syncthreads();
  }
  // The id of the nth occurrence of a value, counted over the CTAs in the order of
  // their slices and inside a CTA over its threads, each with granules in a row.
  __device__ __noinline__ void select(const SpCmd& m) {
    const SpSlice<E> sl = this->sl;
    SpShared& s = sp_shared();
    const int q = (sl.n + SP_NT - 1) / SP_NT;
    const int b = min(sl.n, (int)threadIdx.x * q), e = min(sl.n, b + q);
    int mine = 0;
    for (int i = b; i < e; ++i) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.fetch(i), v);
#pragma unroll
      for (int j = 0; j < SpVec<E>::N; ++j) mine += v[j] == m.value;
    }
    int total;
    int before = sp_block_scan(mine, s.red_i, &total);
    if (threadIdx.x < ranks) of(threadIdx.x).count[rank] = total;
    cl.sync();
    for (int r = 0; r < rank; ++r) before += s.count[r];
    if (m.nth >= before && m.nth < before + mine) {
      int left = m.nth - before;
      for (int i = b; i < e; ++i) {
        float v[SpVec<E>::N];
        SpVec<E>::get(sl.fetch(i), v);
#pragma unroll
        for (int j = 0; j < SpVec<E>::N; ++j)
          if (v[j] == m.value && left-- == 0) of(0).token = sl.id(i, j);
      }
    }
  }
  __device__ __forceinline__ void clear() {
    SpShared& s = sp_shared();
    s.hist4[threadIdx.x] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < SP_SOME / 4) s.some4[threadIdx.x] = make_uint4(0, 0, 0, 0);
  }
  __device__ __noinline__ void carry_out(const SpCmd& m) {
    SpShared& s = sp_shared();
    if (m.op == SP_FIRST) {
      const bool with_k = m.high[SP_K] > -INFINITY, with_m = m.theta > -FLT_MAX;
      if (with_k) with_m ? first_pass<true, true>(m) : first_pass<true, false>(m);
      else with_m ? first_pass<false, true>(m) : first_pass<false, false>(m);
    }
    if (m.op == SP_PASS) pass(m);
    if (m.op == SP_HIST) {
      clear();
      __syncthreads();
      if (m.shift < 0) hist_by_value();
      else hist_by_key(m);
    }
    if (m.op == SP_GATHER) gather(m);
    if (m.op == SP_STREAM) stream(m);
    if (m.op == SP_SELECT) select(m);
  }
  // CTA 0: s.cmd to every CTA, carried out by all; returns when all are done.
  __device__ void command() {
    SpShared& s = sp_shared();
    __syncthreads();
    constexpr int W = sizeof(SpCmd) / 4;
    for (int i = threadIdx.x; i < W * (ranks - 1); i += SP_NT)
      reinterpret_cast<uint32_t*>(&of(1 + i / W).cmd)[i % W] =
          reinterpret_cast<const uint32_t*>(&s.cmd)[i % W];
    cl.sync();
    if (s.cmd.op == SP_DONE) return;
    const SpCmd m = s.cmd;
    carry_out(m);
    cl.sync();
    if (m.op == SP_STREAM) view();
  }
  __device__ void obey() {
    SpShared& s = sp_shared();
    for (;;) {
      cl.sync();
      const SpCmd m = s.cmd;
      if (m.op == SP_DONE) return;
      carry_out(m);
      cl.sync();
      if (m.op == SP_STREAM) view();
    }
  }

  // ---- CTA 0 ----------------------------------------------------------------------
  // The cluster's counts added up: hist4 becomes the counts before each bin, mass
  // about the mass before each bin: n_b times the weight at the bin's centre, or, in the
  // first bins by value, which hold few values and most of the mass, of a value in it.
  template <typename F>
  __device__ __noinline__ int merge(F centre, bool by_value) {
    SpShared& s = sp_shared();
    int n[4] = {0, 0, 0, 0};
    float x[4];
#pragma unroll
    for (int r = 0; r < SP_CLUSTER; ++r)
      if (r < ranks) {
        const uint4 c = of(r).hist4[threadIdx.x];
        const uint4 f = by_value && 4 * threadIdx.x < SP_SOME ? of(r).some4[threadIdx.x]
                                                              : make_uint4(0, 0, 0, 0);
        const uint32_t ci[4] = {c.x, c.y, c.z, c.w};
        const uint32_t fi[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (ci[j]) x[j] = sp_drawn(fi[j]);
          n[j] += (int)ci[j];
        }
      }
    const int b = 4 * threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float rate = (float)k.inv_t;
    float m[4], mi = 0.f;
    int ni = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = !n[j] ? 0.f
             : by_value && b < SP_SOME ? n[j] * __expf((x[j] - k.mx) * rate)
                                       : n[j] * centre(b + j);
      mi += m[j];
      ni += n[j];
    }
    int at = sp_warp_scan(ni), total = 0;
    float ma = sp_warp_scan(mi);
    if (lane == 31) {
      s.red_i[warp] = at;
      s.red_f[warp] = ma;
    }
    __syncthreads();
    at -= ni;
    ma -= mi;
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < SP_NT / 32; ++w) {
      const int c = s.red_i[w];
      const float f = s.red_f[w];
      if (w < warp) {
        at += c;
        ma += f;
      }
      total += c;
      all += f;
    }
    s.hist4[threadIdx.x] = make_uint4(at, at + n[0], at + n[0] + n[1], at + n[0] + n[1] + n[2]);
    *reinterpret_cast<float4*>(&s.mass[b]) = make_float4(ma, ma + m[0], ma + m[0] + m[1], ma + m[0] + m[1] + m[2]);
    if (threadIdx.x == SP_NT - 1) s.mass[SP_BINS] = all;
    __syncthreads();
    return total;
  }
  __device__ __forceinline__ int before(int b, int total) const {
    SpShared& s = sp_shared();
    return b >= SP_BINS ? total : reinterpret_cast<const int*>(s.hist4)[b];
  }
  // The bin of the k-th value (1 <= k <= total).
  __device__ __noinline__ int bin_of_count(int k, int total) {
    SpShared& s = sp_shared();
    for (int b = 4 * threadIdx.x; b < 4 * (int)threadIdx.x + 4; ++b)
      if (before(b, total) < k && k <= before(b + 1, total)) s.got_i = b;
    __syncthreads();
    const int r = s.got_i;
    __syncthreads();
    return r;
  }
  // About the bin where the mass passes m; the last filled bin where none does.
  __device__ __noinline__ int bin_of_mass(float m, int total) {
    SpShared& s = sp_shared();
    if (threadIdx.x == 0) s.got_i = -1;
    __syncthreads();
    for (int b = 4 * threadIdx.x; b < 4 * (int)threadIdx.x + 4; ++b)
      if (s.mass[b] <= m && m < s.mass[b + 1] && before(b, total) < before(b + 1, total))
        atomicMax(&s.got_i, b);
    __syncthreads();
    const int r = s.got_i;
    __syncthreads();
    return r >= 0 ? r : bin_of_count(total, total);
  }
  // A window around bin b: its neighbours too, in [low, high], while they are small
  // (a guess is rarely off by more), the bin alone where it is not.
  __device__ void window_of(int b, int low, int high, int total, int* a, int* z) {
    SpShared& s = sp_shared();
    const int l1 = max(low, b - 1), l2 = max(low, b - 2), h1 = min(high, b + 1), h2 = min(high, b + 2);
    const int up2 = before(l2, total), up1 = before(l1, total), down1 = before(h1 + 1, total),
              down2 = before(h2 + 1, total);
    const bool two = down2 - up2 <= SP_WIDEN, one = down1 - up1 <= SP_RANKED;
    *a = two ? l2 : one ? l1 : b;
    *z = two ? h2 : one ? h1 : b;
  }
  // The largest key whose value falls into bin b or a later one (one below the
  // least finite key where none does): bins are monotone in the value.
  __device__ __noinline__ uint32_t top_of_bin(int b) const {
    SpShared& s = sp_shared();
    uint32_t lo = sp_key(-FLT_MAX) - 1, hi = sp_key(k.mx);
    if (b <= 0) return hi;
    if (b >= SP_BINS) return lo;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (k.bin(sp_value(mid)) >= b) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
  // Sorted list -> this thread's prefix sums and weights, entries i = PER t + j.
  template <int PER>
  __device__ void prefixes(const unsigned long long* list, int n, double* w, double* sum) {
    SpShared& s = sp_shared();
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = PER * threadIdx.x + j;
      w[j] = i < n ? k.weight_any(sp_value((uint32_t)(list[i] >> 32))) : 0.0;
      mine += w[j];
    }
    double all;
    double run = sp_block_scan(mine, s.red_d, &all);
#pragma unroll
    for (int j = 0; j < PER; ++j) sum[j] = run += w[j];
  }
  template <int PER>
  __device__ double sum_at(const double* sum, int i) {
    SpShared& s = sp_shared();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (PER * (int)threadIdx.x + j == i) s.got_d = sum[j];
    __syncthreads();
    const double r = s.got_d;
    __syncthreads();
    return r;
  }
  // How many of the entries satisfy a condition.
  template <int PER, typename F>
  __device__ int count(F holds) {
    SpShared& s = sp_shared();
    if constexpr (PER == 1) return __syncthreads_count(holds(0));
    int n = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) n += holds(j);
    return sp_block_sum(n, s.red_i);
  }
  // All of a row's decisions on the sorted list of its first n values.
  template <int PER>
  __device__ __noinline__ void decide(const SpArgs& a, int row, int n, int wanted, float top_p, float theta, float u) {
    SpShared& s = sp_shared();
    double w[PER], sum[PER];
    prefixes<PER>(s.list, n, w, sum);
    const int i0 = PER * (int)threadIdx.x;
    int many = min(wanted, n);
    if (top_p < 1.0f) {
      const double want = (double)top_p * sum_at<PER>(sum, many - 1);
      many = min(many, count<PER>([&](int j) { return i0 + j < many && sum[j] < want; }) + 1);
    }
    many = count<PER>([&](int j) {
      return i0 + j < many && sp_value((uint32_t)(s.list[i0 + j] >> 32)) >= theta;
    });
    const double left = sum_at<PER>(sum, many - 1);
    const int at = min(count<PER>([&](int j) { return i0 + j < many && sum[j] <= (double)u * left; }),
                       many - 1);
    if (threadIdx.x == 0) {
      const unsigned long long e = s.list[at];
      const double d = ((double)sp_value((uint32_t)(e >> 32)) - (double)k.mx) * k.inv_t;
      sp_write(a, row, (int)(0xFFFFFFFFu - (uint32_t)e), (float)(d - log(left)), many, 0);
    }
  }
};

// A window of values in which a crossing is looked for.
struct SpWindow {
  int a, z;             // its bins (by_key: unused)
  bool by_key;          // found by a histogram of keys inside [klo0, khi0]
  bool weigh;           // a run of bins that does not fit: its own mass is needed too
  uint32_t klo, khi;    // its keys
  uint32_t klo0, khi0;  // by_key: keys between which the crossing is known to lie,
  double above0;        //   and the mass above them
  bool gather;
  SpSpan span;          // the values of which the crossing is one
};

template <typename E>
__global__ void __launch_bounds__(SP_NT, 2) sample_min_p_kernel(const SpArgs a) {
  SpShared& s = sp_shared();
  SpRow<E> R{{}, cg::this_cluster()};
  R.rank = (int)R.cl.block_rank();
  R.ranks = (int)R.cl.num_blocks();
  const int row = blockIdx.x / R.ranks;
  const int t = threadIdx.x;

  // ---- options: the same for every CTA of the row -------------------------------
  SpOptions o;
  if (!o.read(a, row)) {
    if (R.rank == 0 && t == 0) sp_write_bad(a, row, NCB_FLAG_BAD_OPTIONS);
    return;
  }
  const float T = o.T, top_p = o.top_p, min_p = o.min_p, u = o.u;
  const int k_asked = o.top_k;
  const bool greedy = T == 0.0f;

  R.cl.barrier_arrive();  // this CTA runs: the others may write into it
  R.sl.set(static_cast<const E*>(a.logits) + (int64_t)row * a.ld, a.vocab, R.rank, a.per);
  R.T = T;
  R.clear();
  if (t < SP_WINDOWS) s.n_list[t] = 0;
  // ---- maximum, least finite value; where few values are wanted, of a part of the row first --------
  const bool bounded = !greedy && k_asked > 0 && k_asked <= min(SP_BOUNDED, SP_NT * R.ranks / 2);
  bool few = bounded || (!greedy && min_p > 0.0f && top_p >= 1.0f);
  R.part = R.sl.n;
  // (of short slices all: reading them again costs less than sorting more)
  if (few && R.sl.n > 4 * SP_NT)
    R.part = ((k_asked > SP_BOUNDED / 2 ? R.sl.n / 2 : R.sl.n / 4) + SP_NT - 1) / SP_NT * SP_NT;
  float mx = -INFINITY, mn = INFINITY;
  R.sl.template each<4>([&](const float* v, int i) { SpRow<E>::template take<false>(R.sl, v, i, 0.0f, mx, mn); }, 0, R.part);
  float own = mx;
  R.cl.barrier_wait();
  R.share(mx, mn);
  R.cl.sync();
  float top = R.view();
  if (few && top == -INFINITY) {  // nothing there: as if many were wanted
    few = false;
    R.cl.sync();
    R.sl.template each<4>([&](const float* v, int i) { SpRow<E>::template take<false>(R.sl, v, i, 0.0f, mx, mn); }, R.part, R.sl.n);
    R.share(mx, mn);
    R.cl.sync();
    top = R.view();
  }
  if (!R.finite(top)) {
    if (R.rank == 0 && t == 0) sp_write_bad(a, row, NCB_FLAG_NONFINITE);
    return;
  }
  if (greedy) {
    SpCmd m{};
    m.op = SP_SELECT;
    m.value = top;
    R.select(m);
    R.cl.sync();
    if (R.rank == 0 && t == 0) sp_write(a, row, s.token, 0.0f, 1, 0);
    return;
  }

  // ---- few values wanted: those above a bound ------------------------------------------
  // The threads' maxima are so many different values of the row: the bin of the k-th
  // largest of them, or an earlier one, holds the k-th value. The bound comes from the
  // first quarter or half of the row (of which about four or two times k values are
  // above it in the whole row), so that the rest is read once.
  if (few) {
    if (bounded && own > -INFINITY) atomicAdd(reinterpret_cast<int*>(s.hist4) + R.k.bin(own), 1);
    R.cl.sync();
  } else {
    R.hist_by_value();
    R.cl.sync();
  }
  if (R.rank != 0) {
    R.obey();
    return;
  }
  float step;  // nats per bin
  auto centre = [&](int b) { return __expf(-((float)b + 0.5f) * step); };
  if (few) {
    step = 0.0f;
    float least = -FLT_MAX;
    if (bounded) {
      const int maxima = R.merge(centre, false);
      if (maxima >= k_asked) {
        const int deep = R.bin_of_count(k_asked, maxima);
        // not above any value of these bins, whose places are off by 2^-23 of them at most
        const double edge = (double)top - (deep + 1) / (double)R.k.scale * (1.0 + 1e-6);
        if (deep < SP_BINS - 1 && edge > -(double)FLT_MAX) least = nextafterf((float)edge, -INFINITY);
      }
    }
    // the part's maximum is not above the row's, and so is what min-p keeps
    if (t == 0) s.theta = top_p >= 1.0f ? fmaxf(least, sp_least_kept(top, T, min_p, R.k.inv_t)) : least;
    __syncthreads();
    if (t == 0) {
      s.cmd.op = SP_STREAM;
      s.cmd.theta = s.theta;
    }
    R.command();
    top = R.k.mx;
    if (t == 0) s.theta = sp_least_kept(top, T, min_p, R.k.inv_t);
    const int n = s.n_list[0];
    if (!R.finite(top) || n <= SP_FEW) {
      if (t == 0) s.cmd.op = SP_DONE;
      R.command();
      if (!R.finite(top)) {
        if (t == 0) sp_write_bad(a, row, NCB_FLAG_NONFINITE);
        return;
      }
      sp_sort(s.list, n);
      const int k = k_asked > 0 ? k_asked : n;  // (fewer finite values than k: all of them are here)
      if (n <= SP_NT) R.template decide<1>(a, row, n, k, top_p, s.theta, u);
      else R.template decide<SP_FEW / SP_NT>(a, row, n, k, top_p, s.theta, u);
      return;
    }
    if (t == 0) {
      s.cmd.op = SP_HIST;
      s.cmd.shift = -1;
    }
    R.command();
  } else if (t == 0) {
    s.theta = sp_least_kept(top, T, min_p, R.k.inv_t);
  }
  mx = top;
  step = (float)(R.k.inv_t / (double)R.k.scale);
  const int total = R.merge(centre, true);
  const int k = k_asked > 0 && k_asked < total ? k_asked : total;
  const int bk = R.bin_of_count(k, total);
  const float theta = s.theta;  // (written before merge's barriers)
  const int bm = R.k.bin(theta);
  // the last bin that has to be known: all of K where its mass is asked for
  const int deep = top_p < 1.0f ? bk : min(bk, bm);

  if (R.before(deep + 1, total) <= SP_FEW) {
    // ---- few: one list decides ---------------------------------------------------------
    if (t == 0) {
      s.cmd.op = SP_GATHER;
      s.cmd.theta = sp_value(R.top_of_bin(deep + 1) + 1);
      s.n_list[0] = 0;
    }
    R.command();
    if (t == 0) s.cmd.op = SP_DONE;
    R.command();
    const int n = s.n_list[0];
    sp_sort(s.list, n);
    if (n <= SP_NT) R.template decide<1>(a, row, n, k, top_p, theta, u);
    else R.template decide<SP_FEW / SP_NT>(a, row, n, k, top_p, theta, u);
    return;
  }

  // ---- many: exact masses above windows -----------------------------------------------------
  // The guesses, from the counts. K's own crossing needs a window only where K ends
  // before the last finite value.
  const bool by_k = k < total, by_p = top_p < 1.0f;
  const int last = R.bin_of_count(total, total);
  SpWindow win[SP_WINDOWS] = {};
  bool found[SP_WINDOWS] = {!by_k, !by_p, false};
  const float z_guess = by_k ? s.mass[bk] + (s.mass[bk + 1] - s.mass[bk]) *
                                                (float)(k - R.before(bk, total)) /
                                                (float)(R.before(bk + 1, total) - R.before(bk, total))
                             : s.mass[SP_BINS];
  float left_guess = z_guess;
  win[SP_K].a = win[SP_K].z = bk;
  if (by_p) {
    const int b = R.bin_of_mass(top_p * z_guess, total);
    R.window_of(b, 0, last, total, &win[SP_P].a, &win[SP_P].z);
    left_guess = top_p * z_guess;
  }
  if (min_p > 0.0f) left_guess = fminf(left_guess, s.mass[bm] + 0.5f * (s.mass[bm + 1] - s.mass[bm]));
  R.window_of(R.bin_of_mass(u * left_guess, total), 0, last, total, &win[SP_D].a, &win[SP_D].z);

  double mass_k = 0.0, mass_p = 0.0, left = 0.0;  // Z, mass(P), mass(M)
  int n_p = k, many = k;
  bool by_value = true;  // the merged counts are those of the bins of values
  auto need_bins = [&] {
    if (by_value) return;
    if (t == 0) {
      s.cmd.op = SP_HIST;
      s.cmd.shift = -1;
    }
    R.command();
    R.merge(centre, true);
    by_value = true;
  };
  // A window of bins is listed where it fits; then, of all such, the keys.
  auto set_bins = [&](int w) {
    win[w].by_key = win[w].weigh = false;
    win[w].gather = R.before(win[w].z + 1, total) - R.before(win[w].a, total) <= SP_CAP;
  };
  auto set_keys = [&] {
    __syncthreads();
    for (int w = 0; w < SP_WINDOWS; ++w)
      if (!found[w] && !win[w].by_key && (t == 32 * w || t == 32 * w + SP_NT / 2))
        s.tops[t == 32 * w ? w : SP_WINDOWS + w] = R.top_of_bin(t == 32 * w ? win[w].a : win[w].z + 1);
    __syncthreads();
    for (int w = 0; w < SP_WINDOWS; ++w)
      if (!found[w] && !win[w].by_key) {
        win[w].khi = s.tops[w];
        win[w].klo = s.tops[SP_WINDOWS + w] + 1;
      }
  };
  for (int w = 0; w < SP_WINDOWS; ++w) {
    win[w].span = {0, k};  // all three are in K
    if (!found[w]) set_bins(w);
  }

  // After a histogram of the keys in [lo, hi] (whose mass above is `above`, values
  // above n_above): the window around the crossing of `want` (a mass, or a count).
  auto divide = [&](int w, uint32_t lo, uint32_t hi, double above, int n_above, double want,
                    bool count) {
    int shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)SP_BINS) ++shift;
    if (t == 0) {
      s.cmd.op = SP_HIST;
      s.cmd.klo[0] = lo;
      s.cmd.khi[0] = hi;
      s.cmd.shift = shift;
    }
    R.command();
    by_value = false;
    const uint32_t half = shift ? 1u << (shift - 1) : 0u;
    const int n = R.merge([&](int b) {
      const uint32_t key = hi - min(((uint32_t)b << shift) + half, hi - lo);
      return (float)R.k.weight_any(sp_value(key));
    }, false);
    int a1, z1;
    if (count) {
      a1 = z1 = R.bin_of_count((int)want - n_above, n);
    } else {
      const int b = R.bin_of_mass((float)fmax(want - above, 0.0), n);
      R.window_of(b, 0, SP_BINS - 1, n, &a1, &z1);
    }
    win[w].by_key = true;
    win[w].klo0 = lo;
    win[w].khi0 = hi;
    win[w].above0 = above;
    win[w].khi = hi - ((uint32_t)a1 << shift);
    win[w].klo = hi - min((((uint32_t)z1 + 1u) << shift) - 1u, hi - lo);
    win[w].gather = R.before(z1 + 1, n) - R.before(a1, n) <= SP_CAP;
  };

  int token = -1;
  float token_value = 0.0f;
  int nth = -1;  // >= 0: the token is this occurrence of token_value
  // Each turn finds a crossing or excludes values from it for good (sp_turn: a window, or
  // all but one), so the loop ends; the limit is a guard.
  for (int turn = 0; !found[SP_D] && turn < SP_TURNS; ++turn) {
    bool first = true;  // all windows are runs of bins: the first pass will do
    for (int w = 0; w < SP_WINDOWS; ++w) first = first && (found[w] || !(win[w].by_key || win[w].weigh));
    set_keys();
    if (first) need_bins();
    if (t == 0) {
      s.cmd.op = first ? SP_FIRST : SP_PASS;
      s.cmd.theta = theta;
      for (int w = 0; w < SP_WINDOWS; ++w) {
        // a window that is not looked at any more: nothing in it, and above it every
        // value for K (whose mass is then the row's), none for the others
        s.cmd.high[w] = found[w] ? (w == SP_K ? -INFINITY : INFINITY) : sp_edge(win[w].khi);
        s.cmd.low[w] = found[w] ? INFINITY : sp_value(win[w].klo);
        s.cmd.klo[w] = found[w] ? 0xFFFFFFFFu : win[w].klo;
        s.cmd.khi[w] = found[w] ? (w == SP_K ? sp_key(-INFINITY) : sp_key(INFINITY)) : win[w].khi;
        s.cmd.gather[w] = !found[w] && win[w].gather;
        s.n_list[w] = 0;
      }
    }
    R.command();
    SpPart p = s.part[0];
    for (int r = 1; r < R.ranks; ++r) {
#pragma unroll
      for (int j = 0; j < SP_SUMS; ++j) {
        p.mass[j] += s.part[r].mass[j];
        p.n[j] += s.part[r].n[j];
      }
    }
    if (first)  // counts are known; what is in the windows comes with their lists
      for (int w = 0; w < SP_WINDOWS; ++w) {
        if (found[w]) continue;
        p.n[w] = R.before(win[w].a, total);
        p.n[SP_WINDOWS + 1 + w] = R.before(win[w].z + 1, total) - p.n[w];
        if (!win[w].gather) {  // or is one value, or needs its mass from the other pass
          uint32_t low = 0xFFFFFFFFu, high = 0;
          for (int r = 0; r < R.ranks; ++r) {
            low = min(low, s.k_low[r][w]);
            high = max(high, s.k_high[r][w]);
          }
          win[w].klo = low;
          win[w].khi = high;
          p.mass[SP_WINDOWS + 1 + w] = low == high ? p.n_in(w) * R.k.weight_any(sp_value(low)) : -1.0;
        }
      }
    // K ends at the k-th value, counted: its window holds it.
    if (!by_k) {
      mass_k = p.above(SP_K);
    } else if (!found[SP_K]) {
      const int idx = k - p.n_above(SP_K);  // 1 .. n_in
      SpWindow& v = win[SP_K];
      if (v.gather) {
        sp_sort(s.list + SP_K * SP_CAP, p.n_in(SP_K));
        double w[1], sum[1];
        R.template prefixes<1>(s.list + SP_K * SP_CAP, p.n_in(SP_K), w, sum);
        mass_k = p.above(SP_K) + R.template sum_at<1>(sum, idx - 1);
        found[SP_K] = true;
      } else if (v.klo == v.khi) {
        mass_k = p.above(SP_K) + idx * R.k.weight_any(sp_value(v.klo));
        found[SP_K] = true;
      } else {  // (the least and greatest key, or the keys of its bins: k is between them)
        divide(SP_K, v.klo, v.khi, 0.0, p.n_above(SP_K), (double)k, true);
        continue;
      }
    }
    // A crossing of `want` (>=, or > for the draw): 0 found at place *at of the list
    // or of the equal values, 1 the window has moved.
    auto cross = [&](int w, double want, bool beyond, int* at, double* mass) -> int {
      SpWindow& v = win[w];
      const double ab = p.above(w);
      auto past = [&](double x) { return beyond ? x > want : x >= want; };
      const int n = p.n_in(w), above = p.n_above(w);
      const bool up = past(ab) && above > v.span.lo;
      double in = p.in(w), sum[1] = {0.0};
      if (!up && v.gather) {  // the list says what is in the window
        double each[1];
        sp_sort(s.list + w * SP_CAP, n);
        R.template prefixes<1>(s.list + w * SP_CAP, n, each, sum);
        if (first) in = n ? R.template sum_at<1>(sum, n - 1) : 0.0;
      }
      if (first && !v.gather && in < 0.0 && !up) {  // too many different values: their mass first
        v.weigh = true;
        return 1;
      }
      const int way = sp_turn(v.span, above, n, past(ab), past(ab + in));
      const int front = v.span.lo - above, back = v.span.hi - 1 - above;  // SP_HERE: places it may have
      if (way == SP_HERE && v.gather) {
        *at = min(max(R.template count<1>([&](int) { return t < n && !past(ab + sum[0]); }), front), back);
        *mass = ab + R.template sum_at<1>(sum, *at);
        return 0;
      }
      if (way == SP_HERE && v.klo == v.khi) {  // equal values
        const double wt = R.k.weight_any(sp_value(v.klo));
        double j = floor((want - ab) / wt);  // values passed before, give or take one
        if (j > 0.0 && past(ab + j * wt)) j -= 1.0;
        if (!past(ab + (j + 1.0) * wt)) j += 1.0;
        *at = (int)fmin(fmax(j, (double)front), (double)back);
        *mass = ab + (*at + 1.0) * wt;
        return 0;
      }
      if (way != SP_HERE && !v.by_key) {  // the bins just before, or just behind
        need_bins();
        const int b = way == SP_UP ? v.a - 1 : v.z + 1;
        R.window_of(b, way == SP_UP ? 0 : b, way == SP_UP ? b : last, total, &v.a, &v.z);
        set_bins(w);
        return 1;
      }
      const uint32_t lo = way == SP_UP ? v.khi + 1 : way == SP_DOWN ? v.klo0 : v.klo,
                     hi = way == SP_UP ? v.khi0 : way == SP_DOWN ? v.klo - 1 : v.khi;
      divide(w, lo, hi, way == SP_UP ? v.above0 : way == SP_DOWN ? ab + in : ab, 0, want, false);
      return 1;
    };
    int at;
    if (by_p && !found[SP_P]) {
      if (cross(SP_P, (double)top_p * mass_k, false, &at, &mass_p)) continue;
      n_p = p.n_above(SP_P) + at + 1;
      found[SP_P] = true;
    }
    if (!by_p) {
      n_p = k;
      mass_p = mass_k;
    }
    many = n_p;
    left = mass_p;
    if (theta > -FLT_MAX && p.n_above(SP_WINDOWS) < many) {
      many = p.n_above(SP_WINDOWS);
      left = p.above(SP_WINDOWS);
    }
    win[SP_D].span.hi = min(win[SP_D].span.hi, many);
    double unused;
    if (cross(SP_D, (double)u * left, true, &at, &unused)) continue;
    found[SP_D] = true;
    if (win[SP_D].gather) {
      const unsigned long long e = s.list[SP_D * SP_CAP + at];
      token = (int)(0xFFFFFFFFu - (uint32_t)e);
      token_value = sp_value((uint32_t)(e >> 32));
    } else {
      token_value = sp_value(win[SP_D].klo);
      nth = at;
    }
  }
  if (nth >= 0) {
    if (t == 0) {
      s.cmd.op = SP_SELECT;
      s.cmd.value = token_value;
      s.cmd.nth = nth;
    }
    R.command();
    token = s.token;
  }
  if (t == 0) {
    s.cmd.op = SP_DONE;
    if (!found[SP_D]) sp_write_bad(a, row, NCB_FLAG_TIES_OVERFLOW);
  }
  if (t == 0 && found[SP_D]) {
    const double d = ((double)token_value - (double)mx) * R.k.inv_t;
    sp_write(a, row, token, (float)(d - log(left)), many, 0);
  }
  R.command();
}

// ---- rows of 16-bit values ----------------------------------------------------------------
// A 16-bit type has 65536 values, so a row's counts per value say all there is to say
// about it: masses are counts times weights, exact, and there is nothing to guess or
// to sort. One pass counts (a 16-bit counter per value, 128 KiB of shared memory: a
// CTA counts at most 65535 values of the row), one more finds the token's occurrence.
//
// Values are numbered from the greatest down ("places"). Of the merged counts CTA r
// of a cluster owns the r-th part of the places. It writes those that occur down as a
// list of (place, count), which shares the weights out evenly among its threads (the
// places that occur lie close together). A crossing is found by CTA (their totals),
// then by thread (a scan), then by entry.
constexpr int SQ_NT = 1024;
constexpr int SQ_SLICE = 65535;  // values that a CTA may count
constexpr int SQ_ALONE = 32768;  // and that a CTA alone may have: its list takes the counters' place
constexpr int SQ_TILES = SQ_SLICE / 8 / SQ_NT + 2;

struct SqHit {     // where a crossing lies
  int n;           // values kept up to and with it
  int nth;         // which of the place's values it is
  int place;
  double mass;     // of the n values
};
struct SqShared {
  int tot_n[SP_CLUSTER], first[SP_CLUSTER], bad[SP_CLUSTER], kept_n[SP_CLUSTER], here[SP_CLUSTER];
  double tot_m[SP_CLUSTER], kept_m[SP_CLUSTER];  // kept: what min-p keeps
  SqHit hit[SP_WINDOWS];
  int in_warp[SQ_TILES][SQ_NT / 32];  // occurrences of the token's value
  int red_i[SQ_NT / 32], red_j[SQ_NT / 32];
  double red_d[SQ_NT / 32], red_e[SQ_NT / 32];
  float theta;
  int at, last;
};

template <typename E>
struct SqType;
template <>
struct SqType<__nv_bfloat16> {
  static constexpr uint32_t INF = 0x7F80u;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b << 16); }
};
template <>
struct SqType<__half> {
  static constexpr uint32_t INF = 0x7C00u;
  static __device__ __forceinline__ float value(uint32_t b) {
    return __half2float(__ushort_as_half((unsigned short)b));
  }
};
// The bits of the value at a place: +values from the greatest to +0, then -0 to the least.
__device__ __forceinline__ uint32_t sq_bits(int place) {
  return place < 32768 ? 32767u - place : (uint32_t)place;
}

template <typename E, int RANKS>
struct SqRow {
  static constexpr int PLACES = 65536 / RANKS;      // of a CTA
  static constexpr int PAIRS = PLACES / SQ_NT / 2;  // of a thread
  cg::cluster_group cl;
  int rank;
  SpView k;
  int entries, per;        // of the CTA's list, of a thread
  int n, before_n;         // this thread's values, and those before them in the CTA
  double mass, before_m;   // their masses

  // The counters, and then the list: place within the CTA's in the low bits, the count
  // above it (the counts of RANKS slices need as many bits more as the places need
  // fewer).
  static __device__ __forceinline__ uint32_t* counts() { return reinterpret_cast<uint32_t*>(sp_raw); }
  __device__ __forceinline__ int place_of(uint32_t e) const { return rank * PLACES + (int)(e & (PLACES - 1)); }
  static __device__ __forceinline__ int count_of(uint32_t e) { return (int)(e / PLACES); }
  __device__ __forceinline__ double weight(int place) const {
    const float v = SqType<E>::value(sq_bits(place));
    return v >= k.zero ? k.weight(v) : 0.0;
  }
  __device__ __forceinline__ SqShared& of(SqShared& s, int r) const {
    return *cl.map_shared_rank(&s, r);
  }

  // The first value, in the order of the row, that `past` holds for: past(number of
  // values up to it, their mass). Every thread of the cluster calls it; the result is in
  // every CTA's hit[w] after the next cluster barrier.
  template <typename F>
  __device__ void cross(SqShared& s, int w, F past) {
    int owner = -1, base_n = 0, last = 0, last_n = 0;
    double base_m = 0.0, last_m = 0.0;
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      if (owner >= 0) continue;
      if (s.tot_n[r]) last = r, last_n = base_n, last_m = base_m;
      if (s.tot_n[r] && past(base_n + s.tot_n[r], base_m + s.tot_m[r])) {
        owner = r;
      } else {
        base_n += s.tot_n[r];
        base_m += s.tot_m[r];
      }
    }
    if (owner < 0) owner = last, base_n = last_n, base_m = last_m;
    if (owner != rank) return;
    if (threadIdx.x == 0) s.at = SQ_NT, s.last = 0;
    __syncthreads();
    if (n) {
      if (past(base_n + before_n + n, base_m + (before_m + mass))) atomicMin(&s.at, (int)threadIdx.x);
      atomicMax(&s.last, (int)threadIdx.x);
    }
    __syncthreads();
    if ((int)threadIdx.x != (s.at < SQ_NT ? s.at : s.last)) return;
    int bn = base_n + before_n, c = 0, place = 0;
    double bm = base_m + before_m, wt = 0.0;
    const int i0 = threadIdx.x * per, i1 = min(entries, i0 + per);
    for (int i = i0; i < i1; ++i) {
      const uint32_t e = counts()[i];
      place = place_of(e);
      c = count_of(e);
      wt = weight(place);
      if (i == i1 - 1 || past(bn + c, bm + c * wt)) break;
      bn += c;
      bm += c * wt;
    }
    // the least j with past(bn + j + 1, ...)
    int lo = 0, hi = c - 1;
    while (lo < hi) {
      const int j = (lo + hi) / 2;
      if (past(bn + j + 1, bm + (j + 1.0) * wt)) hi = j;
      else lo = j + 1;
    }
    const SqHit h{bn + lo + 1, lo, place, bm + (lo + 1.0) * wt};
#pragma unroll
    for (int r = 0; r < RANKS; ++r) of(s, r).hit[w] = h;
  }
};

template <typename E, int RANKS>
__global__ void __launch_bounds__(SQ_NT, 1) sample_min_p16_kernel(const SpArgs a) {
  __shared__ SqShared s;
  using Row = SqRow<E, RANKS>;
  Row R{cg::this_cluster()};
  R.rank = (int)R.cl.block_rank();
  const int row = blockIdx.x / RANKS, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  SpOptions o;
  if (!o.read(a, row)) {
    if (R.rank == 0 && t == 0) sp_write_bad(a, row, NCB_FLAG_BAD_OPTIONS);
    return;
  }
  const bool greedy = o.T == 0.0f;
  SpSlice<E> sl;
  sl.set(static_cast<const E*>(a.logits) + (int64_t)row * a.ld, a.vocab, R.rank, a.per);

  // ---- counts --------------------------------------------------------------------------
  for (int i = t; i < 8192; i += SQ_NT) sp_raw[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  {
    uint32_t* counts = R.counts();
    constexpr uint32_t none = 0x8000u | SqType<E>::INF;  // -inf
    sl.template each_granule<4, SQ_NT>([&](const uint4& g, int) {
      const uint32_t w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = w[j] & 0xFFFFu, hi = w[j] >> 16;
        if (lo != none) atomicAdd(&counts[lo >> 1], 1u << ((lo & 1) * 16));
        if (hi != none) atomicAdd(&counts[hi >> 1], 1u << ((hi & 1) * 16));
      }
    }, 0, sl.n);
  }
  R.cl.sync();

  // ---- this thread's places, over the cluster ----------------------------------------------------
  // Places 2 m and 2 m + 1 share a counter word; of the positive values the words (and
  // in a word the halves) are in falling order of places. Read by 16 bytes, neighbouring
  // lanes starting at different ones, so that they read different banks (by 4 bytes the
  // other CTAs' words took 20 us).
  constexpr int VECS = Row::PAIRS / 4;
  const int m0 = (R.rank * SQ_NT + t) * Row::PAIRS, turn = lane * VECS / 8;
  const int block = (m0 < 16384 ? 16384 - m0 - Row::PAIRS : m0) / 4;
  int lo[Row::PAIRS], hi[Row::PAIRS];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    uint4* from = sp_raw + block + ((v + turn) & (VECS - 1));
#pragma unroll
    for (int c = 0; c < 4; ++c) lo[4 * v + c] = hi[4 * v + c] = 0;
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      const uint4 x = RANKS == 1 ? *from : *R.cl.map_shared_rank(from, r);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (RANKS == 1) {
          lo[4 * v + c] = (int)w[c];  // both, to be taken apart
        } else {
          lo[4 * v + c] += (int)(w[c] & 0xFFFFu);
          hi[4 * v + c] += (int)(w[c] >> 16);
        }
      }
    }
  }
  const bool down = m0 < 16384;
  auto pair_of = [&](int j) {  // which of the thread's pairs of places it is
    const int q = (((j >> 2) + turn) & (VECS - 1)) * 4 + (j & 3);
    return down ? Row::PAIRS - 1 - q : q;
  };
  auto counts_of = [&](int j, int* c0, int* c1) {
    const int l = RANKS == 1 ? (int)((uint32_t)lo[j] & 0xFFFFu) : lo[j],
              h = RANKS == 1 ? (int)((uint32_t)lo[j] >> 16) : hi[j];
    *c0 = down ? h : l;
    *c1 = down ? l : h;
  };
  unsigned long long filled = 0;  // by place within the thread's
  R.n = 0;
#pragma unroll
  for (int j = 0; j < Row::PAIRS; ++j) {
    if (RANKS == 1 ? lo[j] == 0 : (lo[j] | hi[j]) == 0) continue;
    int c0, c1;
    counts_of(j, &c0, &c1);
    R.n += c0 + c1;
    filled |= (unsigned long long)((c0 ? 1 : 0) | (c1 ? 2 : 0)) << (2 * pair_of(j));
  }
  // Not finite: places of +NaN and +inf come first, those of -NaN last.
  constexpr int P_FIRST = 32768 - (int)SqType<E>::INF, P_LAST = 32768 + (int)SqType<E>::INF - 1;
  const int p0 = 2 * m0;
  int first = 65536, bad = 0;
  if (filled) {
    first = p0 + __ffsll((long long)filled) - 1;
    const int last = p0 + 63 - __clzll((long long)filled);
    bad = first < P_FIRST || last > P_LAST;
  }
  const int nz = __popcll(filled), nz_in = sp_warp_scan(nz);
  {
    const int wn = __reduce_add_sync(0xffffffffu, R.n), wf = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.red_i[warp] = wn, s.in_warp[0][warp] = wf;
    if (lane == 31) s.red_j[warp] = nz_in;
    bad = __syncthreads_or(bad);
    if (t < 32) {
      const int cn = __reduce_add_sync(0xffffffffu, s.red_i[t]),
                cf = __reduce_min_sync(0xffffffffu, s.in_warp[0][t]), nz_w = sp_warp_scan(s.red_j[t]);
      s.in_warp[1][t] = nz_w - s.red_j[t];
      if (t == 31) s.at = nz_w;
      if (t < RANKS) {
        SqShared& to = R.of(s, t);
        to.tot_n[R.rank] = cn;
        to.first[R.rank] = cf;
        to.bad[R.rank] = bad;
      }
    }
    R.cl.sync();  // the counters are not read any more
  }
  int total = 0, top = 65536;
#pragma unroll
  for (int r = 0; r < RANKS; ++r) {
    total += s.tot_n[r];
    top = min(top, s.first[r]);
    bad |= s.bad[r];
  }
  if (bad || total == 0) {
    if (R.rank == 0 && t == 0) sp_write_bad(a, row, NCB_FLAG_NONFINITE);
    return;
  }
  const float mx = SqType<E>::value(sq_bits(top));
  SqHit draw{1, 0, top, 1.0};
  int many = 1;
  double left = 1.0;
  R.k.mx = mx;
  // ---- the list ---------------------------------------------------------------------------------
  R.entries = s.at;
  {
    const int at = s.in_warp[1][warp] + nz_in - nz;
#pragma unroll
    for (int j = 0; j < Row::PAIRS; ++j) {
      if (RANKS == 1 ? lo[j] == 0 : (lo[j] | hi[j]) == 0) continue;
      int c0, c1;
      counts_of(j, &c0, &c1);
      const int b = 2 * pair_of(j);
      const int i = at + __popcll(filled & ((1ull << b) - 1));
      const uint32_t place = (uint32_t)(2 * Row::PAIRS * t + b);
      if (c0) R.counts()[i] = (uint32_t)c0 * Row::PLACES | place;
      if (c1) R.counts()[i + (c0 ? 1 : 0)] = (uint32_t)c1 * Row::PLACES | (place + 1);
    }
  }
  if (!greedy) {
    R.k.inv_t = 1.0 / (double)o.T;
    R.k.c = R.k.inv_t / 0.69314718055994530942;
    const double far = (double)mx - SP_REACH * (double)o.T;
    R.k.zero = far > -(double)FLT_MAX ? (float)far : -FLT_MAX;
    if (t == 0) s.theta = sp_least_kept(mx, o.T, o.min_p, R.k.inv_t);
  }
  __syncthreads();
  if (!greedy) {
    // ---- masses: of this thread's entries, before them, of the CTA's, and what min-p keeps -----------
    R.per = (R.entries + SQ_NT - 1) / SQ_NT;
    const float theta = s.theta;
    R.n = 0;
    R.mass = 0.0;
    int kept_n = 0;
    double kept_m = 0.0;
    for (int i = t * R.per; i < min(R.entries, (t + 1) * R.per); ++i) {
      const uint32_t e = R.counts()[i];
      const int place = R.place_of(e), c = R.count_of(e);
      const double m = c * R.weight(place);
      R.n += c;
      R.mass += m;
      if (SqType<E>::value(sq_bits(place)) >= theta) kept_n += c, kept_m += m;
    }
    const int in = sp_warp_scan(R.n);
    const double im = sp_warp_scan(R.mass);
    kept_n = __reduce_add_sync(0xffffffffu, kept_n);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) kept_m += __shfl_xor_sync(0xffffffffu, kept_m, x);
    if (lane == 31) s.red_i[warp] = in, s.red_d[warp] = im, s.red_j[warp] = kept_n, s.red_e[warp] = kept_m;
    __syncthreads();
    if (t < 32) {
      const int wn = sp_warp_scan(s.red_i[t]);
      const double wm = sp_warp_scan(s.red_d[t]);
      const int kn = __reduce_add_sync(0xffffffffu, s.red_j[t]);
      double km = s.red_e[t];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) km += __shfl_xor_sync(0xffffffffu, km, x);
      if (t == 31)
#pragma unroll
        for (int r = 0; r < RANKS; ++r) {
          SqShared& to = R.of(s, r);
          to.tot_m[R.rank] = wm;
          to.kept_n[R.rank] = kn;
          to.kept_m[R.rank] = km;
        }
      s.red_i[t] = wn - s.red_i[t];
      s.red_d[t] = wm - s.red_d[t];
    }
    __syncthreads();
    R.before_n = s.red_i[warp] + in - R.n;
    R.before_m = s.red_d[warp] + (im - R.mass);
    R.cl.sync();

    // ---- K, P, what min-p keeps, and the draw ------------------------------------------------------
    const int kk = o.top_k > 0 && o.top_k < total ? o.top_k : total;
    int pn = 0;
    double pm = 0.0;
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      left = r ? left + s.tot_m[r] : s.tot_m[r];
      pn += s.kept_n[r];
      pm += s.kept_m[r];
    }
    many = kk;
    if (kk < total) {
      R.cross(s, SP_K, [&](int n, double) { return n >= kk; });
      R.cl.sync();
      left = s.hit[SP_K].mass;
    }
    if (o.top_p < 1.0f) {
      const double want = (double)o.top_p * left;
      R.cross(s, SP_P, [&](int, double x) { return x >= want; });
      R.cl.sync();
      if (s.hit[SP_P].n < many) {
        many = s.hit[SP_P].n;
        left = s.hit[SP_P].mass;
      }
    }
    if (pn < many) many = pn, left = pm;
    const double want = (double)o.u * left;
    R.cross(s, SP_D, [&](int n, double x) { return x > want || n >= many; });
    R.cl.sync();
    draw = s.hit[SP_D];
  }

  // ---- the token: the nth value at the place, by id --------------------------------------------------
  const float value = SqType<E>::value(sq_bits(draw.place));
  int nth = draw.nth;
  if (draw.place == 32768 && !greedy) {  // -0: as good as +0, whose values come before
    __syncthreads();
    if (t == 0) s.at = 0;
    __syncthreads();
    if (R.rank == (32767 / Row::PLACES))
      for (int i = t; i < R.entries; i += SQ_NT)
        if (R.place_of(R.counts()[i]) == 32767) s.at = R.count_of(R.counts()[i]);
    __syncthreads();
    if (RANKS > 1) {
      if (R.rank == (32767 / Row::PLACES) && t < RANKS) R.of(s, t).first[0] = s.at;
      R.cl.sync();
      nth += s.first[0];
    } else {
      nth += s.at;
    }
  }
  const uint32_t want = sq_bits(draw.place), also = value == 0.0f ? want ^ 0x8000u : want;
  auto matches = [&](const uint4& g) {  // bit e: value e of the granule is it
    const uint32_t w[4] = {g.x, g.y, g.z, g.w};
    uint32_t yes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = w[j] & 0xFFFFu, hi = w[j] >> 16;
      yes |= (uint32_t)(lo == want || lo == also) << (2 * j) |
             (uint32_t)(hi == want || hi == also) << (2 * j + 1);
    }
    return yes;
  };
  // tile i of the slice is SQ_NT granules, a warp's part of it 32
  for (int i = warp; i < SQ_TILES; i += SQ_NT / 32) s.in_warp[i][lane] = 0;
  __syncthreads();
  sl.template each_granule<4, SQ_NT>([&](const uint4& g, int i) {
    const uint32_t yes = matches(g);
    if (yes) atomicAdd(&s.in_warp[i / SQ_NT][i % SQ_NT / 32], __popc(yes));
  }, 0, sl.n);
  __syncthreads();
  int mine = 0;  // thread i < SQ_TILES * 32: part i
  if (t < SQ_TILES * 32) mine = s.in_warp[t / 32][t % 32];
  const int inc = sp_warp_scan(mine);
  if (lane == 31) s.red_i[warp] = inc;
  __syncthreads();
  int before = inc - mine, here = 0;
  for (int w = 0; w < SQ_NT / 32; ++w) {
    if (w < warp) before += s.red_i[w];
    here += s.red_i[w];
  }
  if (RANKS > 1) {
    if (t < RANKS) R.of(s, t).here[R.rank] = here;
    R.cl.sync();
    for (int r = 0; r < R.rank; ++r) before += s.here[r];
  }
  if (t == 0) s.at = -1;
  __syncthreads();
  if (mine && nth >= before && nth < before + mine) {
    s.at = t;
    s.last = nth - before;
  }
  __syncthreads();
  if (s.at < 0 || t >= 32) return;
  const int part = s.at * 32 + lane;  // this lane's granule
  const uint32_t yes = part < sl.n ? matches(sl.fetch(part)) : 0;
  const int upto = sp_warp_scan(__popc(yes)), skip = s.last - (upto - __popc(yes));
  if (skip >= 0 && skip < __popc(yes)) {
    uint32_t b = yes;
    for (int i = 0; i < skip; ++i) b &= b - 1;
    const double d = greedy ? 0.0 : ((double)value - (double)mx) * R.k.inv_t;
    sp_write(a, row, sl.id(part, __ffs(b) - 1), (float)(d - log(left)), many, 0);
  }
}

}  // namespace nvs

namespace {

static_assert(sizeof(nvs::SpShared) <= 48 * 1024, "needs no larger limit");
constexpr int SP_DEVICES = 64;

int sp_start(void (*kernel)(nvs::SpArgs), nvs::SpArgs a, int rows, int granules, int ranks,
             int threads, size_t smem, cudaStream_t st) {
  a.per = (granules + ranks - 1) / ranks;
  if ((int64_t)rows * ranks > 0x7FFFFFFFLL) return NCB_ERROR_CAPACITY;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)rows * ranks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? NCB_OK : NCB_ERROR_LAUNCH_FAILED;
}

// A kernel's attribute, set once per device (twice is harmless).
bool sp_once(std::atomic<int>* done, int device, int bit, void (*kernel)(nvs::SpArgs),
             cudaFuncAttribute which, int value) {
  if (device < SP_DEVICES && (done[device].load(std::memory_order_acquire) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, which, value) != cudaSuccess) return false;
  if (device < SP_DEVICES) done[device].fetch_or(bit, std::memory_order_release);
  return true;
}

template <typename E>
int sp_launch(const nvs::SpArgs& a, int rows, int device, int num_sms, cudaStream_t st) {
  // Granules of a row, counting a first one that starts before it.
  const int n = 16 / (int)sizeof(E);
  const int granules = (a.vocab + n - 1) / n + 1;
  if constexpr (sizeof(E) == 2) {
    // as many CTAs to a row as its values need, then as fill the GPU, one per SM
    // (their counters take its shared memory). Each counts up to 65535 values: 128256
    // values need two, which 256 rows' 512 CTAs pay for with 3.5 waves.
    // The options are on the device, so the choice is by size. Counting takes the same
    // time whatever they are; the kernel of the lists, which longer rows take, is faster
    // where few values are wanted and far slower where it has to guess (256x128256 bf16,
    // counts and lists: top_k 50 106 and 49 us, 300 107 and 88, 1000 107 and 179, top_p
    // alone 107 and 1435, greedy 91 and 71).
    const int values = granules * n;
    int ranks = values <= nvs::SQ_ALONE ? 1 : 2;
    while (ranks < nvs::SP_CLUSTER &&
           ((granules + ranks - 1) / ranks * n > nvs::SQ_SLICE ||
            ((int64_t)rows * ranks * 2 <= num_sms && granules / ranks >= 2 * nvs::SQ_NT)))
      ranks *= 2;
    if ((granules + ranks - 1) / ranks * n <= nvs::SQ_SLICE) {
      constexpr int smem = 65536 * 2;
      const auto kernel = ranks == 1   ? nvs::sample_min_p16_kernel<E, 1>
                          : ranks == 2 ? nvs::sample_min_p16_kernel<E, 2>
                          : ranks == 4 ? nvs::sample_min_p16_kernel<E, 4>
                                       : nvs::sample_min_p16_kernel<E, 8>;
      static std::atomic<int> raised[SP_DEVICES];  // a bit per kernel
      if (!sp_once(raised, device, ranks, kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
        return NCB_ERROR_LAUNCH_FAILED;
      return sp_start(kernel, a, rows, granules, ranks, nvs::SQ_NT, smem, st);
    }
  }
  // as many CTAs to a row as fill the GPU twice over, while each has two granules for
  // every thread: a cluster's barriers cost more than they win where rows alone fill
  // it (256x128256: 65 us with one CTA to a row, 81 with two, 119 with four;
  // 1x32000: 27 us with one, 23 with eight)
  int ranks = 1;
  while (ranks < nvs::SP_CLUSTER && (int64_t)rows * ranks * 2 <= 2 * num_sms &&
         granules / ranks >= 2 * nvs::SP_NT)
    ranks *= 2;
  // two CTAs to an SM: without the request the SM was left split for one (89 -> 138 us)
  static std::atomic<int> split[SP_DEVICES];
  if (!sp_once(split, device, 1, nvs::sample_min_p_kernel<E>, cudaFuncAttributePreferredSharedMemoryCarveout, 40))
    return NCB_ERROR_LAUNCH_FAILED;
  return sp_start(nvs::sample_min_p_kernel<E>, a, rows, granules, ranks, nvs::SP_NT,
                  sizeof(nvs::SpShared), st);
}

}  // namespace

extern "C" NCB_API int ncb_sample_rows_min_p_device(
    const void* d_logits, int dtype, int rows, int vocab, int64_t ld, const float* d_uniforms,
    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
    int32_t* d_tokens, float* d_logprobs, int32_t* d_kept, uint32_t* d_flags, void* stream) {
  if (dtype != NCB_DTYPE_F32 && dtype != NCB_DTYPE_F16 && dtype != NCB_DTYPE_BF16)
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows < 0 || vocab <= 0 || ld < vocab) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (rows == 0) return ncb_record_status(NCB_OK);
  if (!d_logits || !d_uniforms || !d_tokens) return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  const uintptr_t low = dtype == NCB_DTYPE_F32 ? 3u : 1u;
  uintptr_t words = 0;
  for (const void* p : {(const void*)d_uniforms, (const void*)d_temperature, (const void*)d_top_k,
                        (const void*)d_top_p, (const void*)d_min_p, (const void*)d_tokens,
                        (const void*)d_logprobs, (const void*)d_kept, (const void*)d_flags})
    words |= reinterpret_cast<uintptr_t>(p);
  if ((reinterpret_cast<uintptr_t>(d_logits) & low) || (words & 3u))
    return ncb_record_status(NCB_ERROR_INVALID_ARGUMENT);
  if (vocab > nvs::SP_MAX_VOCAB) return ncb_record_status(NCB_ERROR_CAPACITY);
  int device = 0, num_sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return ncb_record_status(NCB_ERROR_NO_DEVICE);
  nvs::SpArgs a{};
  a.logits = d_logits;
  a.ld = ld;
  a.vocab = vocab;
  a.uniforms = d_uniforms;
  a.temperature = d_temperature;
  a.top_k = d_top_k;
  a.top_p = d_top_p;
  a.min_p = d_min_p;
  a.tokens = d_tokens;
  a.logprobs = d_logprobs;
  a.kept = d_kept;
  a.flags = d_flags;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int status;
  if (dtype == NCB_DTYPE_F32) status = sp_launch<float>(a, rows, device, num_sms, st);
  else if (dtype == NCB_DTYPE_F16) status = sp_launch<__half>(a, rows, device, num_sms, st);
  else status = sp_launch<__nv_bfloat16>(a, rows, device, num_sms, st);
  return ncb_record_status(status);
}
