// The searches of csrc/sample_search.cuh on the host: what they find, and in how many steps.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <string>
#include <vector>

#include "sample_search.cuh"

static int g_fail = 0, g_run = 0;
#define EXPECT(cond, what)                                                     \
  do {                                                                         \
    ++g_run;                                                                   \
    if (!(cond)) {                                                             \
      ++g_fail;                                                                \
      std::fprintf(stderr, "FAIL %s: %s\n", std::string(what).c_str(), #cond); \
    }                                                                          \
  } while (0)

struct Found {
  float least;
  long steps;
};
static Found least_kept(float mx, float T, float m) {
  long steps = 0;
  const float least = nvs::sp_least_kept(mx, T, m, 1.0 / (double)T, [&] { ++steps; });
  return {least, steps};
}
static bool kept(float v, float mx, float T, float m) {
  return ((double)v - (double)mx) * (1.0 / (double)T) >= std::log((double)m);
}
// The least float that is kept: it is, and its neighbour below is not.
static void check_least(float mx, float T, float m, const char* what) {
  const Found f = least_kept(mx, T, m);
  EXPECT(f.steps <= 100, what);
  EXPECT(f.least <= mx && kept(f.least, mx, T, m), what);
  EXPECT(f.least == -FLT_MAX || !kept(std::nextafterf(f.least, -INFINITY), mx, T, m), what);
}

static void least_kept_tests() {
  // max + T ln m cancels: the floats there are denser than what the difference can tell apart
  check_least(1.83644283f, 0.802564383f, 0.101447009f, "cancels to 1e-17");
  check_least(3.73568249f, 0.967938006f, 0.0210801531f, "cancels to 1e-16");
  EXPECT(least_kept(2.0f, 1.0f, 0.0f).least == -FLT_MAX, "min-p off");
  EXPECT(least_kept(2.0f, 1.0f, 1.0f).least == 2.0f, "only the maximum");
  EXPECT(least_kept(0.0f, 1.0f, 1.0f).least == 0.0f && least_kept(-0.0f, 1.0f, 1.0f).least == 0.0f, "a maximum of 0");
  EXPECT(least_kept(0.0f, FLT_MAX, 1e-45f).least == -FLT_MAX, "everything");
  const float values[] = {0.0f, -0.0f, 1e-45f, -1e-45f, 1.0f, -1.0f, 5.5f, 88.0f, -3e38f, 3.4e38f, 65504.0f, FLT_MAX, -FLT_MAX};
  const float temperatures[] = {1e-45f, 1e-38f, 1e-6f, 0.7f, 1.0f, 1e6f, 3e38f, FLT_MAX};
  const float least_p[] = {1e-45f, 1e-30f, 0.02f, 0.5f, 0.99f, 0.99999994f, 1.0f};
  for (float mx : values)
    for (float T : temperatures)
      for (float m : least_p) check_least(mx, T, m, "extremes");
  std::mt19937_64 g(5);
  std::uniform_real_distribution<double> u(0.0, 1.0);
  long usual = 0;
  for (int i = 0; i < 200000; ++i) {
    const float T = (float)(0.3 + 1.2 * u(g)), m = (float)(0.001 + 0.6 * u(g));
    const float mx = i % 2 ? (float)(20.0 * u(g)) : (float)(-(double)T * std::log((double)m));  // the second: next to 0
    check_least(mx, T, m, "random");
    if (i % 2) usual += least_kept(mx, T, m).steps;
  }
  EXPECT(usual <= 3 * 100000, "an ordinary row takes two or three comparisons");
}

// A search over bins of values as the kernel does it: from a window of bins to its
// neighbour on the side that sp_turn says. `past(n)`: whether the first n values' mass is
// past what is wanted, as one pass has it; it may say something else in the next one.
template <typename F>
static int turns_of(const std::vector<int>& bins, int start, std::mt19937_64& g, F past, nvs::SpSpan* span, int* above,
                    int* in) {
  std::vector<int> before(1, 0);
  for (int n : bins) before.push_back(before.back() + n);
  int a = start, z = start;
  *span = {0, before.back()};
  for (int turn = 1;; ++turn) {
    *above = before[a];
    *in = before[z + 1] - before[a];
    const bool past_above = past(*above), past_through = past(*above + *in);
    const int way = nvs::sp_turn(*span, *above, *in, past_above, past_through);
    if (way == nvs::SP_HERE || turn > 10000) return turn;
    const int wide = (int)(g() % 3);
    if (way == nvs::SP_UP) {
      if (a == 0) return 20000;  // there is nothing
      z = a - 1;
      a = std::max(0, z - wide);
    } else {
      if (z + 1 == (int)bins.size()) return 20000;
      a = z + 1;
      z = std::min((int)bins.size() - 1, a + wide);
    }
  }
}

static void turn_tests() {
  std::mt19937_64 g(9);
  nvs::SpSpan span;
  int above, in;
  // two neighbours that disagree about the edge between them: the lower one decides
  EXPECT(turns_of({5, 7, 6, 4}, 1, g, [&](int n) { return n >= 18 || (n == 12 && above == 12); }, &span, &above, &in) <= 3 &&
             above == 12 && span.lo == 12, "an edge up to rounding");
  for (int i = 0; i < 20000; ++i) {
    std::vector<int> bins(1 + g() % 40);
    int total = 0;
    for (int& n : bins) total += n = g() % 3 ? (int)(g() % 9) : 0;
    if (!total) continue;
    const int start = (int)(g() % bins.size()), wanted = (int)(g() % total);
    // sums that agree: the window that holds the crossing is found
    int turns = turns_of(bins, start, g, [&](int n) { return n > wanted; }, &span, &above, &in);
    EXPECT(turns <= (int)bins.size() && above <= wanted && wanted < above + in && span.lo <= wanted && wanted < span.hi,
           "the crossing's window");
    // sums that agree but for the crossing's own edge, which changes its mind
    turns = turns_of(bins, start, g, [&](int n) { return n == wanted ? g() % 2 == 0 : n > wanted; }, &span, &above, &in);
    EXPECT(turns <= (int)bins.size() + 2 && span.lo <= wanted && wanted <= span.hi, "an edge that changes its mind");
    // whatever the sums say, it ends, in a window with a value that may be it
    turns = turns_of(bins, start, g, [&](int) { return g() % 2 == 0; }, &span, &above, &in);
    EXPECT(turns <= 2 * (int)bins.size() && above <= span.lo && span.lo < span.hi && span.hi <= above + in,
           "any sums");
  }
}

int main() {
  least_kept_tests();
  turn_tests();
  std::printf("%d checks, %d failed\n", g_run, g_fail);
  return g_fail == 0 ? 0 : 1;
}
