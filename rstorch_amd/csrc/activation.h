// The activations of rst_linear_act_* and rst_activation_* (RST_ACT_*), value and derivative, f64.
//
//   relu       max(z, 0)                                   z > 0 ? 1 : 0
//   gelu       z P(z), P(z) = (1 + erf(z / sqrt 2)) / 2    P(z) + z exp(-z^2 / 2) / sqrt(2 pi)
//   gelu_tanh  z s(t), t = 2 sqrt(2 / pi) (z + a z^3)      s + z s (1 - s) t'(z)
//   silu       z s(z), s(t) = 1 / (1 + exp(-t))            s + z s (1 - s)
//
// (z (1 + tanh(t / 2)) / 2 = z s(t): one exponential and a reciprocal instead of a tanh.)  The errors are
// absolute, a few 2^-53 times max(1, |z|).  An infinite z gives the limit (0 or z; derivative 0 or 1)
// rather than the 0 * inf of the formulas; NaN stays NaN, except that relu takes it to 0 as
// rst_relu_forward does.
//
// Inside a contraction kernel every FP64 vector instruction is taken from the matrix cores, which share
// the unit: 8.4 M derivatives of gelu through the library's erf and exp (some 150 instructions) make a
// 480 us pair of products 34 us longer.  So everything here goes through one exponential of a negative
// argument without special cases (16 instructions) and reciprocals without scaling:
//   P(-a) = exp(-a^2 / 2) R(a) for a >= 0, R(a) = exp(a^2 / 2) erfc(a / sqrt 2) / 2 smooth and decaying.  R is
//   a polynomial of degree 13 in u = (69 / 29 a - 6) / (a + 6), which takes [0, 8.7] to [-1, 1]: the minimax
//   fit (in 40 digits) of R weighted with exp(-a^2 / 2), i.e. of P itself; off by 1.3e-17.  The
//   derivative's density is the same exponential.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/rstorch_hip.h"

namespace rst {

constexpr double kGeluTanhScale = 1.5957691216057307117597842397375;  // 2 sqrt(2 / pi)
constexpr double kGeluTanhCube = 0.044715;
constexpr double kActBound = 1e100;  // (its cube is finite; every activation has reached its limit long before)

// 1 / d for a normal d whose reciprocal is normal: the hardware's estimate (24 bits) and two Newton steps.
__device__ __forceinline__ double reciprocal(double d) {
  double y = __builtin_amdgcn_rcp(d);
  y = fma(fma(-d, y, 1.0), y, y);
  return fma(fma(-d, y, 1.0), y, y);
}

// exp(-w) for w >= 0 (0 from w = 746; callers keep w finite): -w = r + n ln 2 with |r| <= ln 2 / 2, minimax
// polynomial of degree 11 in r (3e-18), scaled by 2^n.
__device__ __forceinline__ double exp_minus(double w) {
  const double n = rint(w * -1.4426950408889634);
  double r = fma(n, -0.69314718036912382, -w);  // (the leading 32 bits of ln 2: n times them is exact)
  r = fma(n, -1.9082149292705877e-10, r);
  double p = 2.5118818411059345e-08;
  p = fma(p, r, 2.7632651088911209e-07);
  p = fma(p, r, 2.7557211915565994e-06);
  p = fma(p, r, 2.4801485452468031e-05);
  p = fma(p, r, 0.00019841269924882442);
  p = fma(p, r, 0.0013888888952341407);
  p = fma(p, r, 0.0083333333333012946);
  p = fma(p, r, 0.041666666666488002);
  p = fma(p, r, 0.16666666666666721);
  p = fma(p, r, 0.50000000000000189);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}

// exp(-a^2 / 2) and P(-a) for a in [0, 40] (both 0 from a = 39)
__device__ __forceinline__ void normal_tail(double a, double& density, double& tail) {
  density = exp_minus(0.5 * a * a);
  const double u = fma(a, 2.3793103448275863, -6.0) * reciprocal(a + 6.0);
  double p = -1.5118143999072932e-08;
  p = fma(p, u, -4.4915194709864476e-08);
  p = fma(p, u, 4.450195911249175e-07);
  p = fma(p, u, -8.8861206853693154e-07);
  p = fma(p, u, -1.1125740854421098e-05);
  p = fma(p, u, 0.00012054801263716136);
  p = fma(p, u, -0.00069238778707458133);
  p = fma(p, u, 0.0028740996396699461);
  p = fma(p, u, -0.0094045126049169259);
  p = fma(p, u, 0.025165122414676298);
  p = fma(p, u, -0.055991400257101372);
  p = fma(p, u, 0.1041310995401407);
  p = fma(p, u, -0.16126493282378951);
  p = fma(p, u, 0.14034613460784945);
  tail = density * p;
}

// s(t) = 1 / (1 + exp(-t)) and s (1 - s), neither with a cancellation
__device__ __forceinline__ void logistic(double t, double& s, double& slope) {
  const double e = exp_minus(fmin(fabs(t), 800.0));
  const double q = reciprocal(1.0 + e);
  const double eq = e * q;
  s = t < 0.0 ? eq : q;
  slope = eq * q;
}

__device__ __forceinline__ double gelu_tanh_argument(double z) {
  return kGeluTanhScale * fma(kGeluTanhCube * z * z, z, z);
}

template <int ACT>
__device__ __forceinline__ double act_value(double z) {
  if (ACT == RST_ACT_RELU) return fmax(z, 0.0);
  if (ACT == RST_ACT_NONE) return z;
  z = z < -kActBound ? -kActBound : z;
  if (ACT == RST_ACT_GELU) {
    double density, tail;
    normal_tail(fmin(fabs(z), 40.0), density, tail);
    return z * (z < 0.0 ? tail : 1.0 - tail);
  }
  double s, slope;
  logistic(ACT == RST_ACT_GELU_TANH ? gelu_tanh_argument(z) : z, s, slope);
  return z * s;
}

template <int ACT>
__device__ __forceinline__ double act_gradient(double z) {
  if (ACT == RST_ACT_RELU) return z > 0.0 ? 1.0 : 0.0;
  if (ACT == RST_ACT_NONE) return 1.0;
  z = z < -kActBound ? -kActBound : z;
  z = z > kActBound ? kActBound : z;
  if (ACT == RST_ACT_GELU) {
    double density, tail;
    normal_tail(fmin(fabs(z), 40.0), density, tail);
    return fma(z * 0.39894228040143267794, density, z < 0.0 ? tail : 1.0 - tail);  // 1 / sqrt(2 pi)
  }
  double s, slope;
  logistic(ACT == RST_ACT_GELU_TANH ? gelu_tanh_argument(z) : z, s, slope);
  if (ACT == RST_ACT_GELU_TANH) slope *= kGeluTanhScale * fma(3.0 * kGeluTanhCube * z, z, 1.0);
  return fma(z, slope, s);
}

}  // namespace rst
