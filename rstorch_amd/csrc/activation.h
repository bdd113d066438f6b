// The activations of rst_linear_act_* and rst_activation_* (RST_ACT_*), value and derivative, f64.
//
//   relu       max(z, 0)                                   z > 0 ? 1 : 0
//   gelu       z P(z), P(z) = (1 + erf(z / sqrt 2)) / 2    P(z) + z exp(-z^2 / 2) / sqrt(2 pi)
//   gelu_tanh  z s(t), t = 2 sqrt(2 / pi) (z + a z^3)      s + z s (1 - s) t'(z)
//   silu       z s(z), s(t) = 1 / (1 + exp(-t))            s + z s (1 - s)
//
// (z (1 + tanh(t / 2)) / 2 = z s(t): one exponential and a division instead of a tanh.)  The errors are
// absolute, a few 2^-53 times max(1, |z|): 1 + erf and 1 - s round at 1.  An infinite z gives the
// limit (0 or z; derivative 0 or 1) rather than the 0 * inf of the formulas; NaN stays NaN, except
// that relu takes it to 0 as rst_relu_forward does.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/rstorch_hip.h"

namespace rst {

constexpr double kGeluTanhScale = 1.5957691216057307117597842397375;  // 2 sqrt(2 / pi)
constexpr double kGeluTanhCube = 0.044715;
constexpr double kActBound = 1e100;  // (its cube is finite; every activation has reached its limit long before)

__device__ __forceinline__ double logistic(double t) { return 1.0 / (1.0 + exp(-t)); }

template <int ACT>
__device__ __forceinline__ double act_value(double z) {
  if (ACT == RST_ACT_RELU) return fmax(z, 0.0);
  if (ACT == RST_ACT_NONE) return z;
  z = z < -kActBound ? -kActBound : z;
  if (ACT == RST_ACT_GELU) return 0.5 * z * (1.0 + erf(z * 0.70710678118654752440));
  if (ACT == RST_ACT_GELU_TANH) return z / (1.0 + exp(-kGeluTanhScale * fma(kGeluTanhCube * z * z, z, z)));
  return z / (1.0 + exp(-z));  // silu
}

template <int ACT>
__device__ __forceinline__ double act_gradient(double z) {
  if (ACT == RST_ACT_RELU) return z > 0.0 ? 1.0 : 0.0;
  if (ACT == RST_ACT_NONE) return 1.0;
  z = z < -kActBound ? -kActBound : z;
  z = z > kActBound ? kActBound : z;
  if (ACT == RST_ACT_GELU) {
    const double density = 0.39894228040143267794 * exp(-0.5 * z * z);
    return fma(z, density, 0.5 * (1.0 + erf(z * 0.70710678118654752440)));
  }
  if (ACT == RST_ACT_GELU_TANH) {
    const double zz = z * z;
    const double s = logistic(kGeluTanhScale * fma(kGeluTanhCube * zz, z, z));
    return fma(z * s * (1.0 - s), kGeluTanhScale * fma(3.0 * kGeluTanhCube, zz, 1.0), s);
  }
  const double s = logistic(z);  // silu
  return fma(z * s, 1.0 - s, s);
}

}  // namespace rst
