// The residual-block entry points at the ends of what they accept, over hip_stub.cpp under ASan and UBSan: the stand-in
// refuses a grid that the runtime would, and no arithmetic of a planner overflows.  The address model walks every lane, which
// grids of this size do not allow; here the launches are only counted.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../rstorch_amd/csrc/common.h"
#include "../../rstorch_amd/csrc/gemm_addressing.h"

static long g_shared = 0;  // grids of 32x32 tiles that both gradients of a layer share
void rst::observe_gemm_launch(const rst::GemmLaunch& l) { g_shared += l.kernel == rst::GemmKernel::kStagedMixedGroup; }

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

// a call that is refused before anything is launched
#define REFUSED(expr)                                                                                           \
  do {                                                                                                          \
    const long before_ = hip_stub_launch_count();                                                               \
    const int st_ = (expr);                                                                                     \
    if (st_ != RST_ERR_UNSUPPORTED || hip_stub_launch_count() != before_) {                                     \
      std::fprintf(stderr, "%s:%d: %s -> %d, launched %ld (%s)\n", __FILE__, __LINE__, #expr, st_,              \
                   hip_stub_launch_count() - before_, rst_last_error());                                        \
      std::exit(1);                                                                                             \
    }                                                                                                           \
  } while (0)

static rst_engine* e;
// Operands that lie apart at any size (never dereferenced: kernels do not run)
static double* at(int i) { return reinterpret_cast<double*>((uintptr_t)(i + 1) << 59); }

static int linear(size_t batch, size_t in, size_t out) {
  return rst_linear_act_forward(e, at(0), at(1), at(2), at(3), at(4), at(5), batch, in, out, RST_ACT_SILU);
}

static int backward(size_t batch, size_t in, size_t out, bool need_input = true, int act = RST_ACT_GELU) {
  return rst_linear_act_backward(e, at(0), at(1), act, at(2), at(3), at(4), at(5), at(6), need_input ? at(7) : nullptr, at(8),
                                 RST_ACT_SILU, at(9), batch, in, out);
}
static int plain_backward(size_t batch, size_t in, size_t out, bool need_input = true) {
  return rst_linear_backward(e, at(0), at(3), at(4), at(5), at(6), need_input ? at(7) : nullptr, nullptr, batch, in, out);
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
  }
  // products: fewer than 2^23 tiles of 128x128, which is 2^30 - 128 of one extent while the other fits a tile
  const size_t last = ((size_t)1 << 30) - 128;
  LAUNCHES(linear(last, 1, 1), 1);
  LAUNCHES(linear(last, 100, 128), 1);
  LAUNCHES(linear(9, 1, last), 1);
  LAUNCHES(linear(100, 7, last), 1);
  for (size_t extent : {last + 1, (size_t)1 << 30, ((size_t)1 << 30) + 1}) {
    REFUSED(linear(extent, 1, 1));
    REFUSED(linear(extent, 100, 128));
    REFUSED(linear(9, 1, extent));
    REFUSED(linear(128, 7, extent));
    REFUSED(rst_linear_forward(e, at(0), at(1), at(2), at(5), extent, 1, 1, 0));
  }
  REFUSED(linear((size_t)1 << 29, 5, 129));
  // both gradients: dz and the two products, or nothing
  for (size_t in : {1u, 3u, 128u}) {
    LAUNCHES(backward(last, in, 1), 4);
    REFUSED(backward(last + 1, in, 1));
    REFUSED(backward(1, in, last + 1));
    REFUSED(backward(((size_t)1 << 30) + 1, in, 1));
    REFUSED(backward(9, last + 1, in));
    REFUSED(plain_backward(last + 1, in, 1));
    REFUSED(plain_backward(1, in, last + 1));
  }
  for (size_t batch : {(size_t)500000000, (size_t)700000000, (size_t)749999999})  // a shared grid of 32x32 tiles would not fit
    if (backward(batch, 1, 1) != RST_OK || backward(2, batch, 1) != RST_OK || backward(2, 1, batch) != RST_OK) return 1;
  // (the weight gradient alone is small whatever the batch)
  LAUNCHES(backward(last + 1, 3, 2, false, RST_ACT_NONE), 2);
  LAUNCHES(plain_backward(last + 1, 3, 2, false), 2);
  // the largest extents: refused or run, without an overflow on the way
  for (size_t batch : {9u, 100u, 129u, 5000u}) {
    REFUSED(linear(batch, 1, most));
    REFUSED(linear(most, 1, batch));
    REFUSED(backward(most, batch, 1));
    REFUSED(backward(1, most, batch));
    REFUSED(backward(1, batch, most));
    LAUNCHES(linear(batch, most, 1), 2);
    LAUNCHES(rst_linear_forward(e, at(0), at(1), at(2), at(5), batch, most, 1, 0), 2);
    for (size_t extent : {(size_t)INT_MAX - 1, (size_t)INT_MAX}) {
      REFUSED(rst_linear_forward(e, at(0), at(1), at(2), at(5), batch, 1, extent, 0));
      REFUSED(rst_linear_forward(e, at(0), at(1), at(2), at(5), extent, 1, batch, 0));
      REFUSED(rst_linear_forward(e, at(0), at(1), at(2), at(5), batch, extent, 1, 0));
      REFUSED(plain_backward(extent, batch, 1, false));
      REFUSED(plain_backward(extent, batch, 1));
      REFUSED(plain_backward(1, batch, extent));
    }
  }
  REFUSED(linear(most, most, most));
  // below 1 GFLOP both gradients share a grid, whatever the shape
  const size_t thin[][3] = {{7, 4361, 4431}, {21, 3858, 2909}, {2186, 1794, 62}, {13786, 282, 35}, {3466, 2176, 7}, {22, 1999, 3212},
                            {49, 1225, 3940}, {11550, 1720, 6}, {15896, 482, 29}, {1, 1, 1}, {32, 784, 100}};
  for (auto& d : thin) {
    g_shared = 0;
    if (backward(d[0], d[1], d[2]) != RST_OK || g_shared != 1) {
      std::fprintf(stderr, "%zu rows of %zu -> %zu: %ld shared grids\n", d[0], d[1], d[2], g_shared);
      return 1;
    }
  }
  if (rst_engine_destroy(e) != RST_OK) return 1;
  std::printf("block limits ok\n");
  return 0;
}
