// Sampling with options per row, min-p and 16-bit logits (sm_100a).
//
//   order: x descending, id ascending;  w_i = exp((x_i - max) / T)
//   K = the first top_k of the order, of mass Z;  P = the shortest prefix of K of
//   mass >= top_p Z;  M = {w_i >= min_p} in P;  token = the first of the order
//   whose prefix mass exceeds u mass(M).
//
// Every set is a prefix of the order, so a row needs no sort, only the places
// where a count (top_k), a value (min_p) or a mass (top_p, the draw) is crossed.
// A row belongs to a cluster of 1..8 CTAs, each holding its slice of the row in
// shared memory, so that the row is read from HBM once. CTA 0 decides, the
// others carry out its commands:
//   1. load the slice, maximum and least finite value (NaN and +inf show in a
//      NaN-propagating maximum);
//   2. histogram of counts over SP_BINS equal steps of x below the maximum
//      (counts are integers: their order does not matter). From the counts CTA 0
//      knows the bin of the k-th value exactly, and with n_b exp(centre) about
//      where the masses are crossed;
//   3. few values wanted (the usual options): those bins are gathered into one
//      list, sorted by (x, id), and everything is decided on 64-bit prefix sums
//      of the list. Many: one pass sums the exact 64-bit weights above each
//      guessed window of bins and gathers the windows; a crossing outside its
//      window moves the window and repeats the pass, a window with more values
//      than a list holds is divided by a histogram of the value's bits, down to
//      a single value, whose crossing is a division.
// Sums run in an order fixed by the sizes alone; the lists' order of arrival is
// sorted away.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "navsampler.h"

int ncb_record_status(int st);

namespace nvs {
namespace cg = cooperative_groups;

constexpr int SP_NT = 512;       // threads of a CTA
constexpr int SP_BINS = 2048;    // histogram bins (four per thread)
constexpr int SP_LIST = 2048;    // places of the gather list
constexpr int SP_CAP = 512;      // places of one window's part of it
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

enum { SP_DONE = 0, SP_PASS = 1, SP_HIST = 2, SP_GATHER = 3, SP_SELECT = 4 };
enum { SP_K = 0, SP_P = 1, SP_D = 2, SP_WINDOWS = 3 };

struct SpCmd {
  int op;
  uint32_t klo[SP_WINDOWS], khi[SP_WINDOWS];  // each window's keys, both ends in it
  int gather[SP_WINDOWS];                     // whether its values are listed
  float theta;                                // least value that min-p keeps
  int shift;                                  // SP_HIST: bin = (khi[0] - key) >> shift; < 0: bin(value)
  int bin;                                    // SP_GATHER: bins up to this one
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
  float mass[SP_BINS + 4];   // CTA 0: about the mass before each bin
  unsigned long long list[SP_LIST];
  double table[256];         // 2^(j/256)
  SpCmd cmd;
  SpPart part[SP_CLUSTER];
  float mx[SP_CLUSTER], mn[SP_CLUSTER];
  int count[SP_CLUSTER];
  int n_list[SP_WINDOWS];
  int token;
  int total;  // finite values of the row
  // scratch of the block-wide steps
  double red_d[SP_NT / 32];
  float red_f[SP_NT / 32];
  int red_i[SP_NT / 32];
  SpPart warp_part[SP_NT / 32];
  double got_d;
  int got_i;
  uint32_t tops[8];
};

// Floats in order as unsigned integers; -0 counts as +0.
__device__ __forceinline__ uint32_t sp_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sp_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
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

// A CTA's slice: 16-byte granules [g0, g0 + n) of the row, granule 0 starting at
// the 16-byte boundary at or below the row's first value. Only the row's first and
// last granule can hold values of other rows; they are read value by value and
// filled up with -inf.
template <typename E, bool RES>
struct SpSlice {
  const char* base;  // the row's first granule
  int skip;          // values of granule 0 before the row's first
  int vocab, g0, n;
  uint4* sm;

  __device__ __forceinline__ uint4 fetch(int i) const {
    constexpr int N = SpVec<E>::N;
    const int g = g0 + i;
    const int first = g * N - skip;
    if (first >= 0 && first + N <= vocab)
      return __ldcs(reinterpret_cast<const uint4*>(base) + g);
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
  __device__ __forceinline__ uint4 again(int i) const {
    if constexpr (RES) return sm[i];
    return fetch(i);
  }
  __device__ __forceinline__ int id(int i, int e) const {
    return (g0 + i) * SpVec<E>::N - skip + e;
  }
};

// exp(d c ln2 / 256) for 0 >= d c > -2^20: with d c = n + r, n whole, |r| <= 1/2,
// it is 2^(n / 256) (a table of 2^(j/256) and an exponent) times exp(r ln2 / 256),
// whose series needs four terms for 2^-53. Own code: 64-bit library exponentials
// take about twice the instructions, and a pass over a row is bound by them.
__device__ __forceinline__ double sp_exp(const double* table, double d, double c) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: rounds to a whole number
  constexpr double l = 0.69314718055994530942 / 256.0;
  const double m = d * c;
  const double t = m + magic;
  const double r = m - (t - magic);
  const int n = __double2loint(t);
  const double s = table[n & 255];
  double q = fma(r, l * l * l * l / 24.0, l * l * l / 6.0);
  q = fma(q, r, l * l / 2.0);
  q = fma(q, r, l);
  q = q * r;
  const double w = fma(s, q, s);
  return __hiloint2double(__double2hiint(w) + ((n >> 8) << 20), __double2loint(w));
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

// Bitonic sort, largest first; places [n, power of two) are filled with 0, which
// no listed value has (its low half is never 0).
__device__ void sp_sort(unsigned long long* list, int n) {
  int p = 32;
  while (p < n) p <<= 1;
  for (int i = n + threadIdx.x; i < p; i += SP_NT) list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= p; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int i = threadIdx.x; i < p / 2; i += SP_NT) {
        const int lo = 2 * step * (i / step) + i % step, hi = lo + step;
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

template <typename E, bool RES>
struct SpRow {
  SpShared& s;
  SpSlice<E, RES> sl;
  cg::cluster_group cl;
  int rank, ranks;
  float mx;           // the row's maximum
  double c;           // 256 / (T ln 2)
  double inv_t;
  float scale;        // bins per unit of x
  float zero;         // values below carry no mass (SP_REACH)

  __device__ __forceinline__ int bin(float v) const {
    return min(SP_BINS - 1, __float2int_rd((mx - v) * scale));
  }
  __device__ __forceinline__ double weight(float v) const {
    return sp_exp(s.table, (double)v - (double)mx, c);
  }
  // for listed values, which may lie beyond the reach
  __device__ __forceinline__ double weight_any(float v) const {
    return v < zero ? exp(((double)v - (double)mx) * inv_t) : weight(v);
  }
  __device__ __forceinline__ SpShared& of(int r) { return *cl.map_shared_rank(&s, r); }

  // ---- the commands, carried out by every CTA of the cluster ------------------
  __device__ void hist_by_value() {
    for (int i = threadIdx.x; i < sl.n; i += SP_NT) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.again(i), v);
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e)
        if (v[e] > -INFINITY) atomicAdd(reinterpret_cast<int*>(s.hist4) + bin(v[e]), 1);
    }
  }
  __device__ void hist_by_key(const SpCmd& m) {
    for (int i = threadIdx.x; i < sl.n; i += SP_NT) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.again(i), v);
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e) {
        const uint32_t k = sp_key(v[e]);
        if (k >= m.klo[0] && k <= m.khi[0])
          atomicAdd(reinterpret_cast<int*>(s.hist4) + ((m.khi[0] - k) >> m.shift), 1);
      }
    }
  }
  __device__ __forceinline__ void put(SpShared& to, int w, int base, int cap, float v, int id) {
    const int at = atomicAdd(&to.n_list[w], 1);
    if (at < cap)
      to.list[base + at] = ((unsigned long long)sp_key(v) << 32) | (0xFFFFFFFFu - (uint32_t)id);
  }
  __device__ void gather(const SpCmd& m) {
    SpShared& to = of(0);
    for (int i = threadIdx.x; i < sl.n; i += SP_NT) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.again(i), v);
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e)
        if (v[e] > -INFINITY && bin(v[e]) <= m.bin) put(to, 0, 0, SP_LIST, v[e], sl.id(i, e));
    }
  }
  __device__ void pass(const SpCmd& m) {
    SpShared& to = of(0);
    float lo[SP_WINDOWS], hi[SP_WINDOWS];
#pragma unroll
    for (int w = 0; w < SP_WINDOWS; ++w) {
      lo[w] = sp_value(m.klo[w]);
      // no value has the key of -0; as a float it would take +0 with it
      hi[w] = sp_value(m.khi[w] == 0x7FFFFFFFu ? 0x7FFFFFFEu : m.khi[w]);
    }
    SpPart p{};
    for (int i = threadIdx.x; i < sl.n; i += SP_NT) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.again(i), v);
#pragma unroll
      for (int e = 0; e < SpVec<E>::N; ++e) {
        const float x = v[e];
        if (!(x > -INFINITY)) continue;
        const double wt = x >= zero ? weight(x) : 0.0;
#pragma unroll
        for (int w = 0; w < SP_WINDOWS; ++w) {
          if (x > hi[w]) {
            p.mass[w] += wt;
            ++p.n[w];
          } else if (x >= lo[w]) {
            p.mass[SP_WINDOWS + 1 + w] += wt;
            ++p.n[SP_WINDOWS + 1 + w];
            if (m.gather[w]) put(to, w, w * SP_CAP, SP_CAP, x, sl.id(i, e));
          }
        }
        if (x >= m.theta) {
          p.mass[SP_WINDOWS] += wt;
          ++p.n[SP_WINDOWS];
        }
      }
    }
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
  __device__ void select(const SpCmd& m) {
    const int q = (sl.n + SP_NT - 1) / SP_NT;
    const int b = min(sl.n, (int)threadIdx.x * q), e = min(sl.n, b + q);
    int mine = 0;
    for (int i = b; i < e; ++i) {
      float v[SpVec<E>::N];
      SpVec<E>::get(sl.again(i), v);
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
        SpVec<E>::get(sl.again(i), v);
#pragma unroll
        for (int j = 0; j < SpVec<E>::N; ++j)
          if (v[j] == m.value && left-- == 0) of(0).token = sl.id(i, j);
      }
    }
  }
  __device__ void carry_out(const SpCmd& m) {
    if (m.op == SP_PASS) pass(m);
    if (m.op == SP_HIST) {
      for (int i = threadIdx.x; i < SP_BINS / 4; i += SP_NT) s.hist4[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      if (m.shift < 0) hist_by_value();
      else hist_by_key(m);
    }
    if (m.op == SP_GATHER) gather(m);
    if (m.op == SP_SELECT) select(m);
  }
  // CTA 0: s.cmd to every CTA, carried out by all; returns when all are done.
  __device__ void command() {
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
  }
  __device__ void obey() {
    for (;;) {
      cl.sync();
      const SpCmd m = s.cmd;
      if (m.op == SP_DONE) return;
      carry_out(m);
      cl.sync();
      if (m.op == SP_GATHER) return;  // the last one: CTA 0 has all it needs
    }
  }

  // ---- CTA 0 ----------------------------------------------------------------------
  // The cluster's counts added up: hist4 becomes the counts before each bin, mass
  // about the mass before each bin (n_b times the weight `centre` gives).
  template <typename F>
  __device__ int merge(F centre) {
    uint4 n = make_uint4(0, 0, 0, 0);
    for (int r = 0; r < ranks; ++r) {
      const uint4 x = of(r).hist4[threadIdx.x];
      n.x += x.x;
      n.y += x.y;
      n.z += x.z;
      n.w += x.w;
    }
    const int b = 4 * threadIdx.x;
    const float m0 = n.x ? n.x * centre(b) : 0.f, m1 = n.y ? n.y * centre(b + 1) : 0.f,
                m2 = n.z ? n.z * centre(b + 2) : 0.f, m3 = n.w ? n.w * centre(b + 3) : 0.f;
    int total;
    float all;
    const int at = sp_block_scan((int)(n.x + n.y + n.z + n.w), s.red_i, &total);
    const float ma = sp_block_scan(m0 + m1 + m2 + m3, s.red_f, &all);
    s.hist4[threadIdx.x] = make_uint4(at, at + n.x, at + n.x + n.y, at + n.x + n.y + n.z);
    s.mass[b] = ma;
    s.mass[b + 1] = ma + m0;
    s.mass[b + 2] = ma + m0 + m1;
    s.mass[b + 3] = ma + m0 + m1 + m2;
    if (threadIdx.x == SP_NT - 1) s.mass[SP_BINS] = all;
    __syncthreads();
    return total;
  }
  __device__ __forceinline__ int before(int b, int total) const {
    return b >= SP_BINS ? total : reinterpret_cast<const int*>(s.hist4)[b];
  }
  // The bin of the k-th value (1 <= k <= total).
  __device__ int bin_of_count(int k, int total) {
    for (int b = 4 * threadIdx.x; b < 4 * (int)threadIdx.x + 4; ++b)
      if (before(b, total) < k && k <= before(b + 1, total)) s.got_i = b;
    __syncthreads();
    const int r = s.got_i;
    __syncthreads();
    return r;
  }
  // About the bin where the mass passes m; the last filled bin where none does.
  __device__ int bin_of_mass(float m, int total) {
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
  // The bins around b that one window's list holds: *a .. *z.
  __device__ void window_of(int b, int low, int high, int total, int* a, int* z) {
    *a = *z = b;
    for (int i = 0; i < 16; ++i) {
      if (*a > low && before(*z + 1, total) - before(*a - 1, total) <= SP_CAP) --*a;
      if (*z < high && before(*z + 2, total) - before(*a, total) <= SP_CAP) ++*z;
    }
  }
  // The largest key whose value falls into bin b or a later one (one below the
  // least finite key where none does): bins are monotone in the value.
  __device__ uint32_t top_of_bin(int b) const {
    uint32_t lo = sp_key(-FLT_MAX) - 1, hi = sp_key(mx);
    if (b <= 0) return hi;
    if (b >= SP_BINS) return lo;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (bin(sp_value(mid)) >= b) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
  // Sorted list -> this thread's four prefix sums and weights.
  __device__ void prefixes(const unsigned long long* list, int n, double* w, double* sum) {
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * threadIdx.x + j;
      w[j] = i < n ? weight_any(sp_value((uint32_t)(list[i] >> 32))) : 0.0;
      mine += w[j];
    }
    double all;
    double run = sp_block_scan(mine, s.red_d, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = run += w[j];
  }
  __device__ double sum_at(const double* sum, int i) {
    if (i / 4 == (int)threadIdx.x) s.got_d = sum[i & 3];
    __syncthreads();
    const double r = s.got_d;
    __syncthreads();
    return r;
  }
};

__device__ void sp_write(const SpArgs& a, int row, int token, float logprob, int kept,
                         uint32_t flags) {
  a.tokens[row] = token;
  if (a.logprobs) a.logprobs[row] = logprob;
  if (a.kept) a.kept[row] = kept;
  if (a.flags) a.flags[row] = flags;
}

// A window of values in which a crossing is looked for.
struct SpWindow {
  int a, z;             // its bins (by_key: unused)
  bool by_key;          // found by a histogram of keys inside [klo0, khi0]
  uint32_t klo, khi;    // its keys
  uint32_t klo0, khi0;  // by_key: keys between which the crossing is known to lie,
  double above0;        //   and the mass above them
  bool gather;
};

template <typename E, bool RES>
__global__ void __launch_bounds__(SP_NT, 2) sample_min_p_kernel(const SpArgs a) {
  extern __shared__ uint4 sp_slice[];
  __shared__ SpShared s;
  constexpr int N = SpVec<E>::N;
  SpRow<E, RES> R{s, {}, cg::this_cluster()};
  R.rank = (int)R.cl.block_rank();
  R.ranks = (int)R.cl.num_blocks();
  const int row = blockIdx.x / R.ranks;
  const int t = threadIdx.x;

  // ---- options: the same for every CTA of the row -------------------------------
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const int k_asked = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const float min_p = a.min_p ? a.min_p[row] : 0.0f;
  const float u = a.uniforms[row];
  const bool greedy = T == 0.0f;
  if (!(T >= 0.0f && T <= FLT_MAX) ||
      (!greedy && !(top_p > 0.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f))) {
    if (R.rank == 0 && t == 0)
      sp_write(a, row, -1, __uint_as_float(0x7FC00000u), 0, NCB_FLAG_BAD_OPTIONS);
    return;
  }

  R.cl.barrier_arrive();  // this CTA runs: the others may write into it
  // ---- load, maximum, least finite value ---------------------------------------------
  {
    const char* x = static_cast<const char*>(a.logits) + (int64_t)row * a.ld * (int64_t)sizeof(E);
    R.sl.skip = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(E));
    R.sl.base = x - R.sl.skip * (int)sizeof(E);
    R.sl.vocab = a.vocab;
    const int granules = (a.vocab + R.sl.skip + N - 1) / N;
    R.sl.g0 = min(granules, R.rank * a.per);
    R.sl.n = min(granules, (R.rank + 1) * a.per) - R.sl.g0;
    R.sl.sm = sp_slice;
  }
  if (t < 256) s.table[t] = exp2(t / 256.0);
  for (int i = t; i < SP_BINS / 4; i += SP_NT) s.hist4[i] = make_uint4(0, 0, 0, 0);
  if (t < SP_WINDOWS) s.n_list[t] = 0;
  float mx = -INFINITY, mn = INFINITY;
  {
    constexpr int U = 4;  // loads in flight per thread
    for (int i0 = t; i0 < R.sl.n; i0 += U * SP_NT) {
      uint4 g[U];
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (i0 + j * SP_NT < R.sl.n) g[j] = R.sl.fetch(i0 + j * SP_NT);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (i0 + j * SP_NT < R.sl.n) {
          if constexpr (RES) sp_slice[i0 + j * SP_NT] = g[j];
          float v[N];
          SpVec<E>::get(g[j], v);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            mx = sp_max_nan(mx, v[e]);
            mn = fminf(mn, v[e] == -INFINITY ? INFINITY : v[e]);
          }
        }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = sp_max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if ((t & 31) == 0) {
    s.red_f[t >> 5] = mx;
    s.red_d[t >> 5] = mn;
  }
  __syncthreads();
  R.cl.barrier_wait();
  if (t < R.ranks) {
    for (int w = 0; w < SP_NT / 32; ++w) {
      mx = sp_max_nan(mx, s.red_f[w]);
      mn = fminf(mn, (float)s.red_d[w]);
    }
    R.of(t).mx[R.rank] = mx;
    R.of(t).mn[R.rank] = mn;
  }
  R.cl.sync();
  mx = s.mx[0];
  mn = s.mn[0];
  for (int r = 1; r < R.ranks; ++r) {
    mx = sp_max_nan(mx, s.mx[r]);
    mn = fminf(mn, s.mn[r]);
  }
  if (!(mx >= -FLT_MAX && mx <= FLT_MAX)) {
    if (R.rank == 0 && t == 0)
      sp_write(a, row, -1, __uint_as_float(0x7FC00000u), 0, NCB_FLAG_NONFINITE);
    return;
  }
  R.mx = mx;
  if (greedy) {
    SpCmd m{};
    m.op = SP_SELECT;
    m.value = mx;
    R.select(m);
    R.cl.sync();
    if (R.rank == 0 && t == 0) sp_write(a, row, s.token, 0.0f, 1, 0);
    return;
  }
  R.inv_t = 1.0 / (double)T;
  R.c = 256.0 / 0.69314718055994530942 * R.inv_t;
  // bins over the finite values, as far as they carry mass
  const double far = (double)mx - SP_REACH * (double)T;
  R.zero = far > -(double)FLT_MAX ? (float)far : -FLT_MAX;
  R.scale = (float)((SP_BINS - 1) / ((double)mx - fmax((double)mn, far)));

  // ---- counts ------------------------------------------------------------------------
  R.hist_by_value();
  R.cl.sync();
  if (R.rank != 0) {
    R.obey();
    return;
  }
  const float step = (float)(R.inv_t / (double)R.scale);  // nats per bin
  auto centre = [&](int b) { return __expf(-((float)b + 0.5f) * step); };
  const int total = R.merge(centre);
  const int k = k_asked > 0 && k_asked < total ? k_asked : total;
  // the least value that min-p keeps: w >= m  <=>  x >= max + T ln m
  float theta = -FLT_MAX;
  if (min_p > 0.0f) {
    const double edge = log((double)min_p), least = (double)mx + edge * (double)T;
    theta = least > -(double)FLT_MAX ? (float)least : -FLT_MAX;
    auto kept = [&](float v) { return ((double)v - (double)mx) * R.inv_t >= edge; };
    while (theta < mx && !kept(theta)) theta = nextafterf(theta, INFINITY);
    while (theta > -FLT_MAX && kept(nextafterf(theta, -INFINITY))) theta = nextafterf(theta, -INFINITY);
  }
  const int bk = R.bin_of_count(k, total);
  const int bm = R.bin(theta);
  // the last bin that has to be known: all of K where its mass is asked for
  const int deep = top_p < 1.0f ? bk : min(bk, bm);

  if (R.before(deep + 1, total) <= SP_LIST) {
    // ---- few: one list decides ---------------------------------------------------------
    if (t == 0) {
      s.cmd.op = SP_GATHER;
      s.cmd.bin = deep;
    }
    R.command();
    const int n = s.n_list[0];
    sp_sort(s.list, n);
    double w[4], sum[4];
    R.prefixes(s.list, n, w, sum);
    const int i0 = 4 * t;
    int many = min(k, n);
    if (top_p < 1.0f) {
      const double want = (double)top_p * R.sum_at(sum, many - 1);
      int less = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) less += i0 + j < many && sum[j] < want;
      many = min(many, sp_block_sum(less, s.red_i) + 1);
    }
    int fit = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      fit += i0 + j < many && sp_value((uint32_t)(s.list[min(i0 + j, SP_LIST - 1)] >> 32)) >= theta;
    many = sp_block_sum(fit, s.red_i);
    const double left = R.sum_at(sum, many - 1);
    int passed = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) passed += i0 + j < many && sum[j] <= (double)u * left;
    const int at = min(sp_block_sum(passed, s.red_i), many - 1);
    if (t == 0) {
      const unsigned long long e = s.list[at];
      const double d = ((double)sp_value((uint32_t)(e >> 32)) - (double)mx) * R.inv_t;
      sp_write(a, row, (int)(0xFFFFFFFFu - (uint32_t)e), (float)(d - log(left)), many, 0);
    }
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
    R.merge(centre);
    by_value = true;
  };
  // A window's keys from its bins; its values are listed where they fit.
  auto set_bins = [&](int w) {
    if (t < 2) s.tops[t] = R.top_of_bin(t == 0 ? win[w].a : win[w].z + 1);
    __syncthreads();
    win[w].khi = s.tops[0];
    win[w].klo = s.tops[1] + 1;
    __syncthreads();
    win[w].by_key = false;
    win[w].gather = R.before(win[w].z + 1, total) - R.before(win[w].a, total) <= SP_CAP;
  };
  for (int w = 0; w < SP_WINDOWS; ++w)
    if (!found[w]) set_bins(w);

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
      return (float)R.weight_any(sp_value(key));
    });
    int a1, z1;
    if (count) {
      a1 = z1 = R.bin_of_count((int)want - n_above, n);
    } else {
      const int b = R.bin_of_mass((float)(want - above), n);
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
  // Each turn finds a crossing or leaves it fewer values (a neighbouring window, or
  // the part of one that holds it), so the loop ends; the limit is a guard.
  for (int turn = 0; !found[SP_D] && turn < SP_TURNS; ++turn) {
    if (t == 0) {
      s.cmd.op = SP_PASS;
      s.cmd.theta = theta;
      for (int w = 0; w < SP_WINDOWS; ++w) {
        // a window that is not looked at any more: nothing in it, and above it every
        // value for K (whose mass is then the row's), none for the others
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
    // K ends at the k-th value, counted: its window holds it.
    if (!by_k) {
      mass_k = p.above(SP_K);
    } else if (!found[SP_K]) {
      const int idx = k - p.n_above(SP_K);  // 1 .. n_in
      SpWindow& v = win[SP_K];
      if (v.gather) {
        sp_sort(s.list + SP_K * SP_CAP, p.n_in(SP_K));
        double w[4], sum[4];
        R.prefixes(s.list + SP_K * SP_CAP, p.n_in(SP_K), w, sum);
        mass_k = p.above(SP_K) + R.sum_at(sum, idx - 1);
        found[SP_K] = true;
      } else if (v.klo == v.khi) {
        mass_k = p.above(SP_K) + idx * R.weight_any(sp_value(v.klo));
        found[SP_K] = true;
      } else {
        divide(SP_K, v.klo, v.khi, 0.0, p.n_above(SP_K), (double)k, true);
        continue;
      }
    }
    // A crossing of `want` (>=, or > for the draw): 0 found at place *at of the list
    // or of the equal values, 1 the window has moved.
    auto cross = [&](int w, double want, bool beyond, int* at, double* mass) -> int {
      SpWindow& v = win[w];
      const double ab = p.above(w), in = p.in(w);
      auto past = [&](double x) { return beyond ? x > want : x >= want; };
      const bool here = v.gather || v.klo == v.khi;
      const bool up = past(ab) && p.n_above(w) > 0, down = !up && !past(ab + in);
      if (!up && !down && here) {
        if (v.gather) {
          const unsigned long long* list = s.list + w * SP_CAP;
          const int n = p.n_in(w);
          double wt[4], sum[4];
          sp_sort(s.list + w * SP_CAP, n);
          R.prefixes(list, n, wt, sum);
          int less = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) less += 4 * t + j < n && !past(ab + sum[j]);
          *at = min(sp_block_sum(less, s.red_i), n - 1);
          *mass = ab + R.sum_at(sum, *at);
        } else {
          const double wt = R.weight_any(sp_value(v.klo));
          double j = floor((want - ab) / wt);  // values passed before, give or take one
          if (j > 0.0 && past(ab + j * wt)) j -= 1.0;
          if (!past(ab + (j + 1.0) * wt)) j += 1.0;
          *at = (int)fmin(fmax(j, 0.0), (double)(p.n_in(w) - 1));
          *mass = ab + (*at + 1.0) * wt;
        }
        return 0;
      }
      if (!v.by_key) {
        if (up && v.a > 0) {  // the bins just before
          need_bins();
          const int b = v.a - 1;
          R.window_of(b, 0, b, total, &v.a, &v.z);
          set_bins(w);
        } else if (down && v.z < last) {
          need_bins();
          const int b = v.z + 1;
          R.window_of(b, b, last, total, &v.a, &v.z);
          set_bins(w);
        } else {
          divide(w, v.klo, v.khi, ab, p.n_above(w), want, false);
        }
        return 1;
      }
      if (up && v.khi < v.khi0) divide(w, v.khi + 1, v.khi0, v.above0, 0, want, false);
      else if (down && v.klo > v.klo0) divide(w, v.klo0, v.klo - 1, ab + in, 0, want, false);
      else divide(w, v.klo, v.khi, ab, p.n_above(w), want, false);
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
    if (p.n_above(SP_WINDOWS) < many) {
      many = p.n_above(SP_WINDOWS);
      left = p.above(SP_WINDOWS);
    }
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
    if (!found[SP_D]) sp_write(a, row, -1, __uint_as_float(0x7FC00000u), 0, NCB_FLAG_TIES_OVERFLOW);
  }
  if (t == 0 && found[SP_D]) {
    const double d = ((double)token_value - (double)mx) * R.inv_t;
    sp_write(a, row, token, (float)(d - log(left)), many, 0);
  }
  R.command();
}

}  // namespace nvs

namespace {

// The dynamic shared memory a CTA may hold its slice in, per kernel and device
// (raised once; setting it twice is harmless).
constexpr int SP_DEVICES = 64;
constexpr int SP_MAX_SLICE = 184 * 1024;  // of 227 KiB, beside SpShared

template <typename E, bool RES>
int sp_launch(const nvs::SpArgs& a, int rows, int ranks, size_t smem, int device, cudaStream_t st) {
  auto kernel = nvs::sample_min_p_kernel<E, RES>;
  static std::atomic<bool> raised[SP_DEVICES];
  if (RES && !raised[device].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SP_MAX_SLICE) !=
        cudaSuccess)
      return NCB_ERROR_LAUNCH_FAILED;
    raised[device].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)rows * ranks);
  cfg.blockDim = dim3(nvs::SP_NT);
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

template <typename E>
int sp_dispatch(nvs::SpArgs a, int rows, int device, cudaStream_t st) {
  // Granules of a row, counting a first one that starts before it.
  const int n = 16 / (int)sizeof(E);
  const int granules = (a.vocab + n - 1) / n + 1;
  int ranks = 1;
  // as many CTAs as fill the GPU, while each has work for its threads; then as many
  // as let two CTAs share an SM
  while (ranks < nvs::SP_CLUSTER && (int64_t)rows * ranks * 2 <= 296 && granules / ranks >= 512)
    ranks *= 2;
  while (ranks < nvs::SP_CLUSTER && (int64_t)granules * 16 / ranks > 72 * 1024) ranks *= 2;
  a.per = (granules + ranks - 1) / ranks;
  const size_t smem = (size_t)a.per * 16;
  if ((int64_t)rows * ranks > 0x7FFFFFFFLL) return NCB_ERROR_CAPACITY;
  if (smem <= (size_t)SP_MAX_SLICE) return sp_launch<E, true>(a, rows, ranks, smem, device, st);
  return sp_launch<E, false>(a, rows, ranks, 0, device, st);
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
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= SP_DEVICES)
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
  if (dtype == NCB_DTYPE_F32) status = sp_dispatch<float>(a, rows, device, st);
  else if (dtype == NCB_DTYPE_F16) status = sp_dispatch<__half>(a, rows, device, st);
  else status = sp_dispatch<__nv_bfloat16>(a, rows, device, st);
  return ncb_record_status(status);
}
