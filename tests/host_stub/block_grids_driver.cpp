// Both gradients of a layer in one grid, over hip_stub.cpp with every lane's addresses checked by the address model
// (address_model.cpp): the shapes whose grids block_ops_driver.cpp does not reach.
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "../../include/rstorch_hip.h"

extern "C" long hip_stub_launch_count();

static double* at(int i) { return reinterpret_cast<double*>((uintptr_t)(i + 1) << 44); }

int main() {
  rst_engine* e = nullptr;
  if (rst_engine_create(0, &e) != RST_OK) return 1;
  auto launches = [&](size_t batch, size_t in, size_t out, size_t odd) {  // odd: addresses that are not 16-byte aligned
    const long before = hip_stub_launch_count();
    const int st = rst_linear_act_backward(e, at(0) + odd, nullptr, RST_ACT_NONE, nullptr, at(3) + odd, at(4) + odd, at(5) + odd,
                                           at(6) + odd, at(7) + odd, at(8) + odd, RST_ACT_GELU, at(9) + odd, batch, in, out);
    if (st != RST_OK) {
      std::fprintf(stderr, "%zu rows of %zu -> %zu: %d (%s)\n", batch, in, out, st, rst_last_error());
      std::exit(1);
    }
    return hip_stub_launch_count() - before;
  };
  for (size_t odd = 0; odd < 2; ++odd) {
    // 128x128 tiles, the input gradient's first (it has as many or fewer), the weight gradient's first
    const size_t pairs[][3] = {{1024, 4096, 2000}, {1024, 4096, 1024}, {1023, 4095, 1111}, {1000, 4090, 1025}, {2064, 2048, 2046}, {1111, 4095, 1023}};
    for (auto& d : pairs)
      if (launches(d[0], d[1], d[2], odd) != 1) {
        std::fprintf(stderr, "%zu rows of %zu -> %zu are not one launch\n", d[0], d[1], d[2]);
        return 1;
      }
    // 32x32 tiles of a thin product beside a wide one
    const size_t thin[][3] = {{7, 4361, 4431}, {21, 3858, 2909}, {2186, 1794, 62}, {13786, 282, 35}, {3466, 2176, 7}};
    for (auto& d : thin) launches(d[0], d[1], d[2], odd);
  }
  if (rst_engine_destroy(e) != RST_OK) return 1;
  std::printf("block grids ok\n");
  return 0;
}
