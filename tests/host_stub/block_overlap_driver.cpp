// rst_linear_act_forward / _backward with one array over another, over hip_stub.cpp: every pair of an output and another
// array, at the same address, shifted by one element and end to end.  Accepted is what the header allows, the rest is refused
// before anything is launched.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../../include/rstorch_hip.h"

extern "C" long hip_stub_launch_count();

static rst_engine* e;
static int failures = 0;
constexpr size_t B = 24, K = 10, N = 6;  // batch, in, out

static void expect(bool accepted, int status, long launched, const char* what, const char* out, const char* in, int how) {
  const bool right = accepted ? status == RST_OK && launched > 0 : status == RST_ERR_INVALID_ARGUMENT && launched == 0;
  if (right) return;
  std::fprintf(stderr, "%s: %s over %s (%s): status %d, %ld launches\n", what, out, in,
               how == 0 ? "the same address" : how == 1 ? "one element further" : how == 2 ? "one element before its end" : "behind it",
               status, launched);
  ++failures;
}

struct Arrays {
  double* p[10];
};
static Arrays apart() {
  Arrays a;
  for (int i = 0; i < 10; ++i) a.p[i] = reinterpret_cast<double*>((uintptr_t)(i + 1) << 40);
  return a;
}

// where `out` begins: how 0 at in, 1 one element further, 2 at its last element, 3 right behind it
static double* place(double* in, size_t count, int how) { return in + (how == 0 ? 0 : how == 1 ? 1 : how == 2 ? count - 1 : count); }

enum { GRAD, PRE, X, W, IPRE, RES, GPRE, GW, GB, GI };
static const char* const kNames[] = {"grad", "pre", "x", "weight", "input_pre", "residual_grad", "grad_pre", "grad_weight", "grad_bias", "grad_input"};
static const size_t kCounts[] = {B * N, B * N, B * K, N * K, B * K, B * K, B * N, N * K, N, B * K};

static int backward(const Arrays& a, bool act, bool input_act, bool need_input) {
  return rst_linear_act_backward(e, a.p[GRAD], a.p[PRE], act ? RST_ACT_GELU : RST_ACT_NONE, a.p[GPRE], a.p[X], a.p[W], a.p[GW], a.p[GB],
                                 need_input ? a.p[GI] : nullptr, a.p[IPRE], input_act ? RST_ACT_SILU : RST_ACT_NONE, a.p[RES], B, K, N);
}

static void check_backward(bool act, bool input_act, bool need_input, const char* what) {
  // is the array read or written by this call at all, and is it still when the products run?
  auto used = [&](int i) {
    if (i == PRE || i == GPRE) return act;
    if (i == IPRE) return input_act && need_input;
    if (i == W || i == RES || i == GI) return need_input;
    return true;
  };
  auto late = [&](int i) { return used(i) && !(act && (i == GRAD || i == PRE)); };
  auto may_be = [&](int out, int in) {  // at the same address
    if (out == GPRE) return in == GRAD || in == PRE;
    return out == GI && (in == IPRE || in == RES);
  };
  for (int out = GPRE; out <= GI; ++out)
    for (int in = GRAD; in <= GI; ++in) {
      if (in == out || !used(out)) continue;
      for (int how = 0; how < 4; ++how) {
        Arrays a = apart();
        a.p[out] = place(a.p[in], kCounts[in], how);
        bool ok = how == 3 || !used(in);
        if (out != GPRE) ok = ok || !late(in);
        if (how == 0 && used(in) && may_be(out, in)) ok = true;
        const long before = hip_stub_launch_count();
        const int st = backward(a, act, input_act, need_input);
        expect(ok, st, hip_stub_launch_count() - before, what, kNames[out], kNames[in], how);
      }
    }
}

static int forward(double* const* p, size_t k) {  // x, weight, bias, residual, pre_out, out
  return rst_linear_act_forward(e, p[0], p[1], p[2], p[3], p[4], p[5], B, k, N, RST_ACT_GELU);
}

int main() {
  if (rst_engine_create(0, &e) != RST_OK) return 1;
  check_backward(true, true, true, "an activation on either side");
  check_backward(true, false, true, "an activation behind");
  check_backward(false, true, true, "an activation in front");
  check_backward(false, false, true, "no activation");
  check_backward(true, true, false, "an activation behind, no input gradient");
  check_backward(false, false, false, "no activation, no input gradient");
  {
    // the block in place: one gradient is the skipped one and where the result goes, dz lies apart ...
    Arrays a = apart();
    a.p[RES] = a.p[GI] = a.p[GRAD];
    a.p[GPRE] = a.p[PRE];
    long before = hip_stub_launch_count();
    expect(true, backward(a, true, true, true), hip_stub_launch_count() - before + 1, "in place", "grad_input", "grad", 0);
    // ... and not over it: the skipped gradient would be dz
    a = apart();
    a.p[RES] = a.p[GPRE] = a.p[GRAD];
    before = hip_stub_launch_count();
    int st = backward(a, true, true, true);
    expect(false, st, hip_stub_launch_count() - before, "the skipped gradient is grad", "grad_pre", "grad", 0);
    // operands that are read only may be one array
    a = apart();
    a.p[IPRE] = a.p[X];
    a.p[RES] = a.p[GRAD];
    before = hip_stub_launch_count();
    st = backward(a, true, true, true);
    expect(true, st, hip_stub_launch_count() - before, "operands that are one array", "input_pre", "x", 0);
  }
  const char* const names[] = {"x", "weight", "bias", "residual", "pre_out", "out"};
  for (size_t k : {K, (size_t)0}) {
    const size_t counts[] = {B * k, N * k, N, B * N, B * N, B * N};
    for (int out = 4; out < 6; ++out)
      for (int in = 0; in < 6; ++in)
        for (int how = 0; how < 4; ++how) {
          if (in == out || counts[in] == 0) continue;
          Arrays a = apart();
          a.p[out] = place(a.p[in], counts[in], how);
          const long before = hip_stub_launch_count();
          const int st = forward(a.p, k);
          expect(how == 3 || (how == 0 && out == 5 && in == 3), st, hip_stub_launch_count() - before, k ? "forward" : "forward, no features in",
                 names[out], names[in], how);
        }
  }
  if (rst_engine_destroy(e) != RST_OK || failures) return 1;
  std::printf("block overlap ok\n");
  return 0;
}
