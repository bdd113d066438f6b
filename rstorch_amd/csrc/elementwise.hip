// HBM-bound passes of the residual block: activations (value and derivative, each with an optional
// residual) and dropout.  Every array is read once and written once in 16-byte accesses.
#include <cmath>

#include "activation.h"
#include "common.h"
#include "counter_rng.h"
#include "vec.h"

namespace rst {
namespace {

// One pair per thread, as in the other streaming kernels; a grid has at most 2^31 threads, and longer
// arrays are walked with that stride.
constexpr int kBlock = 64;
constexpr size_t kMaxBlocks = (size_t)1 << 25;

// Calls body(i, two) for every pair [i, i + 2) of [0, n); two == false for the odd last element.
template <class Body>
__device__ __forceinline__ void for_each_pair(size_t n, Body body) {
  const size_t stride = 2 * (size_t)gridDim.x * kBlock;
  for (size_t i = 2 * ((size_t)blockIdx.x * kBlock + threadIdx.x); i < n; i += stride) body(i, i + 1 < n);
}

unsigned blocks_for(size_t n) {
  const size_t blocks = (n + 2 * kBlock - 1) / (2 * kBlock);
  return (unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

// out = act(z) [+ residual].  16384 x 4096: ReLU 160 us (6.7 TB/s, as a flat copy), SiLU 170, tanh GELU 173; GELU 194: its
// normal tail takes as many vector instructions as the bytes take time.
template <int ACT, bool RES>
__global__ __launch_bounds__(kBlock) void act_forward_kernel(const double* z, const double* residual, double* out,
                                                             size_t n) {
  for_each_pair(n, [&](size_t i, bool two) {
    if (two) {
      const v2u v = load2_stream(z + i);
      v2u r;
      r.x = act_value<ACT>(v.x);
      r.y = act_value<ACT>(v.y);
      if (RES) r += load2_stream(residual + i);
      store2(out + i, r);
    } else {
      const double r = act_value<ACT>(z[i]);
      out[i] = RES ? r + residual[i] : r;
    }
  });
}

// out = g * act'(z) [+ residual]; with ACT == NONE z is not read.  16384 x 4096: 247 us (6.5 TB/s), GELU 274.
template <int ACT, bool RES>
__global__ __launch_bounds__(kBlock) void act_backward_kernel(const double* g, const double* z, const double* residual,
                                                              double* out, size_t n) {
  for_each_pair(n, [&](size_t i, bool two) {
    if (two) {
      v2u r = load2_stream(g + i);
      if (ACT != RST_ACT_NONE) {
        const v2u v = load2_stream(z + i);
        r.x *= act_gradient<ACT>(v.x);
        r.y *= act_gradient<ACT>(v.y);
      }
      if (RES) r += load2_stream(residual + i);
      store2(out + i, r);
    } else {
      double r = g[i];
      if (ACT != RST_ACT_NONE) r *= act_gradient<ACT>(z[i]);
      out[i] = RES ? r + residual[i] : r;
    }
  });
}

// Dropout: element i is kept when the generator's value(seed, stream, i) >= p, i.e. when the top 53
// bits of its word are at least ceil(p 2^53); the backward pass draws the same words again.  A dropped
// element is 0 whatever x holds there (inf and NaN included).  A mask that is drawn again costs two 64-bit multiplies an
// element and no bytes: 16384 x 4096 162 us (6.6 TB/s), 2047 x 4095 with a residual 32 us (6.2 TB/s).
template <bool RES>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const double* x, const double* residual, double* out, size_t n,
                                                         uint64_t key, uint64_t threshold, double scale) {
  for_each_pair(n, [&](size_t i, bool two) {
    const bool keep0 = (draw(key, i) >> 11) >= threshold;
    if (two) {
      const bool keep1 = (draw(key, i + 1) >> 11) >= threshold;
      const v2u v = load2_stream(x + i);
      v2u r;
      r.x = keep0 ? v.x * scale : 0.0;
      r.y = keep1 ? v.y * scale : 0.0;
      if (RES) r += load2_stream(residual + i);
      store2(out + i, r);
    } else {
      const double r = keep0 ? x[i] * scale : 0.0;
      out[i] = RES ? r + residual[i] : r;
    }
  });
}

template <int ACT>
void act_forward(hipStream_t s, const double* z, const double* residual, double* out, size_t n) {
  if (residual)
    hipLaunchKernelGGL((act_forward_kernel<ACT, true>), dim3(blocks_for(n)), dim3(kBlock), 0, s, z, residual, out, n);
  else
    hipLaunchKernelGGL((act_forward_kernel<ACT, false>), dim3(blocks_for(n)), dim3(kBlock), 0, s, z, residual, out, n);
}

template <int ACT>
void act_backward(hipStream_t s, const double* g, const double* z, const double* residual, double* out, size_t n) {
  if (residual)
    hipLaunchKernelGGL((act_backward_kernel<ACT, true>), dim3(blocks_for(n)), dim3(kBlock), 0, s, g, z, residual, out,
                       n);
  else
    hipLaunchKernelGGL((act_backward_kernel<ACT, false>), dim3(blocks_for(n)), dim3(kBlock), 0, s, g, z, residual, out,
                       n);
}

}  // namespace

int launch_act_forward(hipStream_t s, int activation, const double* z, const double* residual, double* out, size_t n) {
  if (n == 0) return RST_OK;
  switch (activation) {
    case RST_ACT_RELU: act_forward<RST_ACT_RELU>(s, z, residual, out, n); break;
    case RST_ACT_GELU: act_forward<RST_ACT_GELU>(s, z, residual, out, n); break;
    case RST_ACT_GELU_TANH: act_forward<RST_ACT_GELU_TANH>(s, z, residual, out, n); break;
    case RST_ACT_SILU: act_forward<RST_ACT_SILU>(s, z, residual, out, n); break;
    default: act_forward<RST_ACT_NONE>(s, z, residual, out, n); break;
  }
  RST_HIP(hipGetLastError());
  return RST_OK;
}

int launch_act_backward(hipStream_t s, int activation, const double* g, const double* z, const double* residual,
                        double* out, size_t n) {
  if (n == 0) return RST_OK;
  switch (activation) {
    case RST_ACT_RELU: act_backward<RST_ACT_RELU>(s, g, z, residual, out, n); break;
    case RST_ACT_GELU: act_backward<RST_ACT_GELU>(s, g, z, residual, out, n); break;
    case RST_ACT_GELU_TANH: act_backward<RST_ACT_GELU_TANH>(s, g, z, residual, out, n); break;
    case RST_ACT_SILU: act_backward<RST_ACT_SILU>(s, g, z, residual, out, n); break;
    default: act_backward<RST_ACT_NONE>(s, g, z, residual, out, n); break;
  }
  RST_HIP(hipGetLastError());
  return RST_OK;
}

int launch_dropout(hipStream_t s, const double* x, const double* residual, double* out, size_t n, double p,
                   uint64_t seed, uint64_t stream) {
  if (n == 0) return RST_OK;
  const uint64_t key = tensor_key(seed, stream);
  const uint64_t threshold = (uint64_t)std::ceil(std::ldexp(p, 53));  // (scaling by a power of two is exact)
  const double scale = 1.0 / (1.0 - p);
  if (residual)
    hipLaunchKernelGGL(dropout_kernel<true>, dim3(blocks_for(n)), dim3(kBlock), 0, s, x, residual, out, n, key,
                       threshold, scale);
  else
    hipLaunchKernelGGL(dropout_kernel<false>, dim3(blocks_for(n)), dim3(kBlock), 0, s, x, residual, out, n, key,
                       threshold, scale);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

}  // namespace rst
