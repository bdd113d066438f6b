// The residual-block entry points, built for the host against hip_stub.cpp under ASan and UBSan:
// every refusal comes back as its status before anything is launched, and every accepted shape gets
// through the planners (kernels do not run).  The stand-in aborts on an allocation or a synchronisation
// during stream capture, which covers "nothing here allocates or waits".
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdint>
#include <cstdlib>
#include <initializer_list>
#include <limits>

#include "../../include/rstorch_hip.h"

extern "C" long hip_stub_launch_count();
extern "C" long hip_stub_allocation_calls();
extern "C" void hip_stub_begin_capture(void* stream);
extern "C" int hip_stub_end_capture(void* stream);

static long g_launches = 0;
// a call with the status it has to return; a refusal launches nothing
#define EXPECT(expr, want)                                                                                    \
  do {                                                                                                        \
    g_launches = hip_stub_launch_count();                                                                     \
    int st_ = (expr);                                                                                         \
    if (st_ != (want) || ((want) != RST_OK && hip_stub_launch_count() != g_launches)) {                       \
      std::fprintf(stderr, "%s:%d: %s -> %d, expected %d (%s)\n", __FILE__, __LINE__, #expr, st_, (int)(want), \
                   rst_last_error());                                                                         \
      std::exit(1);                                                                                           \
    }                                                                                                         \
  } while (0)
#define LAUNCHES(expr, count)                                                                             \
  do {                                                                                                    \
    const long before_ = hip_stub_launch_count();                                                         \
    EXPECT(expr, RST_OK);                                                                                 \
    if (hip_stub_launch_count() - before_ != (count)) {                                                   \
      std::fprintf(stderr, "%s:%d: %s launched %ld kernels, expected %d\n", __FILE__, __LINE__, #expr,     \
                   hip_stub_launch_count() - before_, (int)(count));                                       \
      std::exit(1);                                                                                       \
    }                                                                                                     \
  } while (0)

int main() {
  rst_engine* e = nullptr;
  EXPECT(rst_engine_create(0, &e), RST_OK);
  double* const p = reinterpret_cast<double*>((uintptr_t)1 << 40);  // never dereferenced: kernels do not run
  double *const q = p + ((size_t)1 << 36), *const r = q + ((size_t)1 << 36);
  // (of an accepted backward pass: outputs that are no operand)
  double *const x = r + ((size_t)1 << 36), *const w = x + ((size_t)1 << 36), *const gw = w + ((size_t)1 << 36);
  double *const gb = gw + ((size_t)1 << 36), *const ip = gb + ((size_t)1 << 36), *const res = ip + ((size_t)1 << 36);
  double* const none = nullptr;
  const double nan = std::nan(""), inf = std::numeric_limits<double>::infinity();
  const size_t huge = (size_t)1 << 31;
  const int INVALID = RST_ERR_INVALID_ARGUMENT, SHAPE = RST_ERR_SHAPE, UNSUPPORTED = RST_ERR_UNSUPPORTED;

  // layer norm
  EXPECT(rst_layer_norm_forward(nullptr, p, p, p, p, p, p, 4, 4, 1e-5), INVALID);
  EXPECT(rst_layer_norm_forward(e, none, p, p, p, p, p, 4, 4, 1e-5), INVALID);
  EXPECT(rst_layer_norm_forward(e, p, p, p, none, p, p, 4, 4, 1e-5), INVALID);
  for (double eps : {-1e-5, nan, inf}) EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, 4, 4, eps), INVALID);
  EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, 4, 0, 1e-5), SHAPE);
  EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, huge, 4, 1e-5), UNSUPPORTED);
  EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, 4, huge, 1e-5), UNSUPPORTED);
  LAUNCHES(rst_layer_norm_forward(e, none, none, none, none, none, none, 0, 4, 1e-5), 0);
  LAUNCHES(rst_layer_norm_forward(e, p, none, none, p, none, none, 4, 4, 0.0), 1);
  EXPECT(rst_layer_norm_backward(nullptr, p, p, p, p, p, p, p, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, none, p, p, p, p, p, p, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, none, p, p, p, p, p, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, p, p, none, p, p, p, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, none, p, p, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, none, p, p, 4, 4), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, 0, 4), SHAPE);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, 4, 0), SHAPE);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, huge, 4), UNSUPPORTED);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, 4, huge), UNSUPPORTED);
  // two row sums per row and the strips' column sums share the scratch
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, (size_t)9 << 20, 20000), UNSUPPORTED);
  for (size_t cols : {1u, 10u, 60u, 100u, 200u, 400u, 1000u, 2000u, 4096u, 8192u, 8193u, 16384u, 16385u, 32768u, 3000001u, 9000001u})
    for (size_t rows : {1u, 2u, 31u, 1000u, 100000u}) {
      EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, rows, cols, 1e-5), RST_OK);
      EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, rows, cols), RST_OK);
    }

  // dropout
  for (double bad : {-0.1, 1.0, 1.5, nan, inf}) {
    EXPECT(rst_dropout_forward(e, p, p, p, 8, bad, 1, 2), INVALID);
    EXPECT(rst_dropout_backward(e, p, p, 8, bad, 1, 2), INVALID);
  }
  EXPECT(rst_dropout_forward(nullptr, p, p, p, 8, 0.5, 1, 2), INVALID);
  EXPECT(rst_dropout_forward(e, none, p, p, 8, 0.5, 1, 2), INVALID);
  EXPECT(rst_dropout_forward(e, p, p, none, 8, 0.5, 1, 2), INVALID);
  EXPECT(rst_dropout_backward(e, none, p, 8, 0.5, 1, 2), INVALID);
  EXPECT(rst_dropout_backward(e, p, none, 8, 0.5, 1, 2), INVALID);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, none, p, p, p, ((size_t)1 << 23) + 1, 1), UNSUPPORTED);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, none, p, p, p, (size_t)1 << 23, 1), RST_OK);
  LAUNCHES(rst_dropout_forward(e, none, none, none, 0, 0.5, 1, 2), 0);
  LAUNCHES(rst_dropout_forward(e, p, none, p, 1, 0.0, 1, 2), 1);
  LAUNCHES(rst_dropout_backward(e, p, p, (size_t)1 << 36, std::nextafter(1.0, 0.0), 1, 2), 1);

  // activations
  for (int bad : {-1, 5, 1000}) {
    EXPECT(rst_activation_forward(e, p, p, p, 8, bad), INVALID);
    EXPECT(rst_activation_backward(e, p, p, p, p, 8, bad), INVALID);
    EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, 8, 8, 8, bad), INVALID);
    EXPECT(rst_linear_act_backward(e, p, p, bad, p, p, p, p, p, q, p, RST_ACT_NONE, p, 8, 8, 8), INVALID);
    EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_NONE, p, p, p, p, p, q, p, bad, p, 8, 8, 8), INVALID);
  }
  EXPECT(rst_activation_forward(e, none, p, p, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_activation_forward(e, p, p, none, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_activation_backward(e, none, p, p, p, 8, RST_ACT_SILU), INVALID);
  EXPECT(rst_activation_backward(e, p, none, p, p, 8, RST_ACT_SILU), INVALID);
  EXPECT(rst_activation_backward(e, p, p, p, none, 8, RST_ACT_SILU), INVALID);
  LAUNCHES(rst_activation_backward(e, p, none, p, p, 8, RST_ACT_NONE), 1);
  LAUNCHES(rst_activation_forward(e, none, none, none, 0, RST_ACT_RELU), 0);

  // Linear with activation and residual
  EXPECT(rst_linear_act_forward(nullptr, p, p, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, none, p, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, none, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, p, p, p, r, none, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, huge, 8, 8, RST_ACT_GELU), UNSUPPORTED);
  EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, 8, huge, 8, RST_ACT_GELU), UNSUPPORTED);
  EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, 8, 8, huge, RST_ACT_GELU), UNSUPPORTED);
  // no features in: out = act(bias) + residual, nothing to multiply
  LAUNCHES(rst_linear_act_forward(e, none, none, p, p, r, q, 8, 0, 8, RST_ACT_GELU), 1);
  LAUNCHES(rst_linear_act_forward(e, none, none, p, p, r, q, 2, 0, 8, RST_ACT_GELU), 1);
  // the tiles' row and column numbers stay below 2^31
  for (size_t most : {(size_t)INT_MAX, (size_t)INT_MAX - 126}) {
    EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, most, 1, 1, RST_ACT_GELU), UNSUPPORTED);
    EXPECT(rst_linear_act_forward(e, p, p, p, p, r, q, 1, 1, most, RST_ACT_GELU), UNSUPPORTED);
    EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, p, p, p, q, p, RST_ACT_GELU, p, 1, most, 1), UNSUPPORTED);
    EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, most, 2, 0.1), UNSUPPORTED);
  }
  // an output over an operand that is still read
  EXPECT(rst_linear_act_forward(e, q, p, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, q, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, r, p, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, r, p, p, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, p, p, r, r, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, p, p, p, q, q, 8, 8, 8, RST_ACT_GELU), INVALID);
  EXPECT(rst_linear_act_forward(e, p, p, p, q, r, q, 8, 8, 8, RST_ACT_GELU), RST_OK);
  LAUNCHES(rst_linear_act_forward(e, none, none, none, none, none, none, 0, 8, 8, RST_ACT_GELU), 0);
  EXPECT(rst_linear_act_backward(e, none, p, RST_ACT_GELU, p, p, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, none, RST_ACT_GELU, p, p, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, none, p, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, none, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, none, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, p, none, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, p, p, p, q, none, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  for (int zero = 0; zero < 3; ++zero)
    EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, p, p, p, q, p, RST_ACT_GELU, p, zero == 0 ? 0 : 8,
                                   zero == 1 ? 0 : 8, zero == 2 ? 0 : 8), SHAPE);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, p, p, p, q, p, RST_ACT_GELU, p, huge, 8, 8), UNSUPPORTED);
  EXPECT(rst_linear_act_backward(e, p, none, RST_ACT_NONE, none, p, p, gw, none, none, none, RST_ACT_GELU, none, 8, 8, 8), RST_OK);
  // grad_input over x, the weight, or the gradient that both products read
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, q, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, p, q, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, q, p, p, p, p, q, p, RST_ACT_GELU, p, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, q, p, RST_ACT_GELU, q, p, p, p, p, q, p, RST_ACT_GELU, q, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, q, none, RST_ACT_NONE, none, p, p, p, p, q, none, RST_ACT_NONE, q, 8, 8, 8), INVALID);
  EXPECT(rst_linear_act_backward(e, q, p, RST_ACT_GELU, p, x, w, gw, gb, q, ip, RST_ACT_GELU, q, 8, 8, 8), RST_OK);

  // inside a stream capture, over the routes of the planner
  const long allocations = hip_stub_allocation_calls();
  hip_stub_begin_capture(rst_engine_stream(e));
  for (size_t b : {1u, 3u, 8u, 9u, 33u, 512u, 2048u})
    for (size_t k : {1u, 100u, 785u, 4096u})
      for (size_t n : {1u, 10u, 101u, 1024u, 4608u})
        for (int act = RST_ACT_NONE; act <= RST_ACT_SILU; ++act) {
          EXPECT(rst_linear_act_forward(e, p, p, p, act & 1 ? p : none, act & 2 ? r : none, q, b, k, n, act), RST_OK);
          EXPECT(rst_linear_act_backward(e, p, p, act, p, x, w, gw, gb, q, ip, RST_ACT_SILU - act, act & 1 ? res : none, b, k, n), RST_OK);
        }
  // slices of one gradient, of the other, of both, in the shared grid
  const size_t shared[][3] = {{1157, 233, 203}, {46, 2607, 939}, {518, 3, 2177}, {1953, 32, 3607}, {314, 1467, 790}, {2500, 20, 20}};
  for (auto& d : shared)
    EXPECT(rst_linear_act_backward(e, p, p, RST_ACT_GELU, p, x, w, gw, gb, q, ip, RST_ACT_GELU, res, d[0], d[1], d[2]), RST_OK);
  EXPECT(rst_layer_norm_forward(e, p, p, p, p, p, p, 100, 1000, 1e-5), RST_OK);
  EXPECT(rst_layer_norm_backward(e, p, p, p, p, p, p, p, p, p, 100, 1000), RST_OK);
  EXPECT(rst_dropout_forward(e, p, p, p, 100, 0.5, 1, 2), RST_OK);
  if (hip_stub_end_capture(rst_engine_stream(e)) <= 0) { std::fprintf(stderr, "nothing was recorded\n"); return 1; }
  if (hip_stub_allocation_calls() != allocations) { std::fprintf(stderr, "an operator allocated\n"); return 1; }
  EXPECT(rst_engine_destroy(e), RST_OK);
  std::printf("block ops ok\n");
  return 0;
}
