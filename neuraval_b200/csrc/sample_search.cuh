// The searches of the sampling with options per row (sample_min_p.cu) that need no GPU:
// plain functions of numbers, compiled for the host too, so that how many steps they
// take can be tested there.
#pragma once

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>

#ifdef __CUDACC__
#define NVS_BOTH __host__ __device__ __forceinline__
#else
#define NVS_BOTH inline
#endif

namespace nvs {

NVS_BOTH uint32_t sp_bits(float v) {
#ifdef __CUDA_ARCH__
  return __float_as_uint(v);
#else
  uint32_t b;
  std::memcpy(&b, &v, 4);
  return b;
#endif
}
NVS_BOTH float sp_float(uint32_t b) {
#ifdef __CUDA_ARCH__
  return __uint_as_float(b);
#else
  float v;
  std::memcpy(&v, &b, 4);
  return v;
#endif
}
// Floats in order as unsigned integers; -0 counts as +0.
NVS_BOTH uint32_t sp_key(float v) {
  const uint32_t b = sp_bits(v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
NVS_BOTH float sp_value(uint32_t k) { return sp_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// The least key of [bottom, top] for which `holds`, which holds for `top` and, where it
// holds, for all greater keys. Looked for from `guess` on in steps of 1, 2, 4 .., then by
// halves: two questions where the guess is right, 64 and a few at most.
template <typename F>
NVS_BOTH uint32_t sp_least_key(uint32_t bottom, uint32_t top, uint32_t guess, F holds) {
  uint32_t lo, hi, step = 1;  // in the end: not holding, holding
  if (holds(guess)) {
    for (hi = guess;; step = step < 0x80000000u ? 2 * step : step) {
      if (hi == bottom) return bottom;
      lo = hi - (step < hi - bottom ? step : hi - bottom);
      if (!holds(lo)) break;
      hi = lo;
    }
  } else {
    for (lo = guess;; step = step < 0x80000000u ? 2 * step : step) {
      hi = lo + (step < top - lo ? step : top - lo);
      if (hi == top || holds(hi)) break;
      lo = hi;
    }
  }
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (holds(mid)) hi = mid;
    else lo = mid;
  }
  return hi;
}

// The least value that min-p keeps: w >= m  <=>  x >= max + T ln m, compared as (x - max) / T
// in 64 bits. The guess is off by a float or so, except where max + T ln m is next to 0:
// there the floats are so dense that (x - max) rounds to the same for up to 2^30 of them.
// `count` sees every comparison.
template <typename C>
NVS_BOTH float sp_least_kept(float mx, float T, float min_p, double inv_t, C count) {
  if (!(min_p > 0.0f)) return -FLT_MAX;
  const double edge = log((double)min_p), at = fma(edge, (double)T, (double)mx);
  float guess = at > -(double)FLT_MAX ? (float)at : -FLT_MAX;
  guess = guess < mx ? guess : mx;
  return 0.0f + sp_value(sp_least_key(sp_key(-FLT_MAX), sp_key(mx), sp_key(guess), [&](uint32_t k) {
           count();
           return ((double)sp_value(k) - (double)mx) * inv_t >= edge;
         }));
}

// A crossing of a mass is looked for in windows, runs of values in the order. The mass
// above a window and that of the values in it are sums of their own, added up in
// another order than its neighbour's: where the crossing is an edge between two windows
// up to rounding, the upper one may say that it is below and the lower one that it is
// above. So what a window has said stays: the crossing is one of the values lo .. hi - 1
// of the order, which only become fewer.
struct SpSpan {
  int lo, hi;
};
enum { SP_HERE, SP_UP, SP_DOWN };
// Which way from a window of `in` values behind `above` others: past_above, past_through:
// whether the mass above it, and with it, is past what is wanted. SP_HERE: the crossing
// is one of the window's values (at least one of which is in the span then). SP_UP and
// SP_DOWN exclude the window, and there are values on that side.
NVS_BOTH int sp_turn(SpSpan& s, int above, int in, bool past_above, bool past_through) {
  const int end = above + in;
  if (in == 0) past_through = past_above;  // an empty window is never the place
  if (past_above && above > s.lo) {
    if (above < s.hi) s.hi = above;
    return SP_UP;
  }
  if (!past_through && end < s.hi) {
    if (end > s.lo) s.lo = end;
    return SP_DOWN;
  }
  if (end <= s.lo) return SP_DOWN;
  if (above >= s.hi) return SP_UP;
  if (above > s.lo) s.lo = above;
  if (end < s.hi) s.hi = end;
  return SP_HERE;
}

}  // namespace nvs
