// The residual-block entry points at the ends of what they accept, over hip_stub.cpp under ASan and UBSan: the stand-in
// refuses a grid that the runtime would, and no arithmetic of a planner overflows.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../include/rstorch_hip.h"

extern "C" long hip_stub_launch_count();

// a call that is accepted and launches `count` kernels
#define LAUNCHES(expr, count)                                                                                   \
  do {                                                                                                          \
    const long before_ = hip_stub_launch_count();                                                               \
    const int st_ = (expr);                                                                                     \
    const long got_ = hip_stub_launch_count() - before_;                                                        \
    if (st_ != RST_OK || got_ != (long)(count)) {                                                               \
      std::fprintf(stderr, "%s:%d: %s -> %d with %ld launches, expected %ld (%s)\n", __FILE__, __LINE__, #expr, st_, got_, \
                   (long)(count), rst_last_error());                                                            \
      std::exit(1);                                                                                             \
    }                                                                                                           \
  } while (0)

static rst_engine* e;
// Operands that lie apart at any size (never dereferenced: kernels do not run)
static double* at(int i) { return reinterpret_cast<double*>((uintptr_t)(i + 1) << 44); }

static int linear(size_t batch, size_t in, size_t out) {
  return rst_linear_act_forward(e, at(0), at(1), at(2), at(3), at(4), at(5), batch, in, out, RST_ACT_SILU);
}

int main() {
  if (rst_engine_create(0, &e) != RST_OK) return 1;
  const size_t most = (size_t)INT_MAX - 127;

  // a few rows: four features per workgroup of 256 threads, 2^25 features per launch
  for (size_t batch : {1u, 2u, 3u, 4u, 5u, 8u}) {
    LAUNCHES(linear(batch, 1, ((size_t)1 << 25) - 3), 1);
    LAUNCHES(linear(batch, 1, (size_t)1 << 25), 1);
    LAUNCHES(linear(batch, 1, ((size_t)1 << 25) + 1), 2);
    LAUNCHES(linear(batch, 1, ((size_t)1 << 26) - 4), 2);
    LAUNCHES(linear(batch, 1, (size_t)1 << 26), 2);
    LAUNCHES(linear(batch, 1, 100000000), 3);
    LAUNCHES(linear(batch, 1, most), 64);
    LAUNCHES(linear(batch, most, 1), 1);
    LAUNCHES(linear(batch, most, most), 64);
  }
  if (rst_engine_destroy(e) != RST_OK) return 1;
  std::printf("block limits ok\n");
  return 0;
}
