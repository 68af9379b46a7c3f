// The searches of csrc/sample_search.cuh on the host: what they find, and in how many steps.
#include <cmath>
#include <cstdio>
#include <random>
#include <string>

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

int main() {
  least_kept_tests();
  std::printf("%d checks, %d failed\n", g_run, g_fail);
  return g_fail == 0 ? 0 : 1;
}
