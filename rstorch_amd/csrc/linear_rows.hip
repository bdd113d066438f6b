// Linear forward for a few rows (inference one sample at a time): out = act(x w^T + bias) + residual with
// x[rows, k], rows <= 8.
//
// The weights are read once, 8 bytes for 2 rows flops: bound by HBM, and a 32x32 or 64x64 tile of a matrix
// kernel would multiply mostly padding while too few of its loads are in flight.  Here a wavefront takes
// kFeatures weight rows and streams its share of their length in 16-byte loads, 1 KiB of a row each, a batch
// of them in flight; a lane multiplies its pair of weights with the same pair of every x row (x is small and
// stays in the caches).  The wavefronts of a workgroup share the length of the same weight rows; their sums
// meet in LDS and are added in wavefront order, then the epilogue runs.
// 4096 -> 4096 features: one row 23 us (5.8 TB/s; 30.5 on the tiles), eight rows 34 (42 on the tiles).
#include "activation.h"
#include "common.h"
#include "vec.h"

namespace rst {
namespace {

constexpr int kFeatures = 4;  // weight rows per workgroup

// pairs k, k + 1 of a row of n values, 0 beyond the end; any address
template <bool STREAM>
__device__ __forceinline__ v2u pair_or_zero(const double* row, size_t k, size_t n) {
  v2u v = {0.0, 0.0};
  if (k + 1 < n) v = STREAM ? load2_stream(row + k) : load2(row + k);
  else if (k < n) v.x = row[k];
  return v;
}

__device__ __forceinline__ double activate(int activation, double z) {
  switch (activation) {
    case RST_ACT_RELU: return act_value<RST_ACT_RELU>(z);
    case RST_ACT_GELU: return act_value<RST_ACT_GELU>(z);
    case RST_ACT_GELU_TANH: return act_value<RST_ACT_GELU_TANH>(z);
    case RST_ACT_SILU: return act_value<RST_ACT_SILU>(z);
    default: return z;
  }
}

// ROWS: rows of x, rounded up to a power of two (rows beyond the real ones repeat the last and are not
// stored); WAVES wavefronts per workgroup; DEPTH steps of 128 values in flight; `begin_feature`: the launch's first.
template <int ROWS, int WAVES, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void linear_rows_kernel(const double* __restrict__ x,
                                                                 const double* __restrict__ w,
                                                                 const double* __restrict__ bias, double* out,
                                                                 const ActEpilogue e, int rows, size_t features,
                                                                 size_t length, size_t begin_feature) {
  constexpr int VALUES = ROWS * kFeatures;
  constexpr int LOG = VALUES == 4 ? 2 : VALUES == 8 ? 3 : VALUES == 16 ? 4 : 5;
  static_assert(VALUES == 1 << LOG, "four to thirty-two sums");
  __shared__ double part[WAVES][VALUES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t first = begin_feature + (size_t)blockIdx.x * kFeatures;
  const double* wr[kFeatures];
  const double* xr[ROWS];
#pragma unroll
  for (int f = 0; f < kFeatures; ++f) wr[f] = w + (first + f < features ? first + f : features - 1) * length;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) xr[r] = x + (size_t)(r < rows ? r : rows - 1) * length;
  // this wavefront's steps of 128 values: [begin, end)
  const size_t steps = (length + 127) / 128, share = (steps + WAVES - 1) / WAVES;
  const size_t begin = wave * share < steps ? wave * share : steps;
  const size_t end = begin + share < steps ? begin + share : steps;
  double sum[VALUES];
#pragma unroll
  for (int i = 0; i < VALUES; ++i) sum[i] = 0.0;
  auto multiply = [&](const v2u (&wv)[kFeatures], const v2u (&xv)[ROWS]) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int f = 0; f < kFeatures; ++f) {
        sum[r * kFeatures + f] = fma(wv[f].x, xv[r].x, sum[r * kFeatures + f]);
        sum[r * kFeatures + f] = fma(wv[f].y, xv[r].y, sum[r * kFeatures + f]);
      }
  };
  size_t s = begin;
  // whole batches of whole steps (the very last step of a row may be cut short)
  const size_t whole = end * 128 <= length ? end : end - (end > begin ? 1 : 0);
  for (; s + DEPTH <= whole; s += DEPTH) {
    v2u wv[DEPTH][kFeatures], xv[DEPTH][ROWS];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const size_t k = (s + d) * 128 + 2 * lane;
#pragma unroll
      for (int f = 0; f < kFeatures; ++f) wv[d][f] = load2_stream(wr[f] + k);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) xv[d][r] = load2(xr[r] + k);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) multiply(wv[d], xv[d]);
  }
  for (; s < end; ++s) {
    v2u wv[kFeatures], xv[ROWS];
    const size_t k = s * 128 + 2 * lane;
#pragma unroll
    for (int f = 0; f < kFeatures; ++f) wv[f] = pair_or_zero<true>(wr[f], k, length);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) xv[r] = pair_or_zero<false>(xr[r], k, length);
    multiply(wv, xv);
  }
  // Sums over the lanes: every exchange halves the number of sums a lane carries, so that lane l ends up
  // with sum l >> (6 - LOG) of half the remaining lanes; the last exchanges complete it.
#pragma unroll
  for (int n = VALUES / 2, off = 32; n > 0; n /= 2, off /= 2) {
    const bool upper = (lane & off) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const double give = upper ? sum[i] : sum[i + n];
      const double keep = upper ? sum[i + n] : sum[i];
      sum[i] = keep + __shfl_xor(give, off);
    }
  }
#pragma unroll
  for (int off = 32 >> LOG; off > 0; off /= 2) sum[0] += __shfl_xor(sum[0], off);
  if ((lane & ((64 >> LOG) - 1)) == 0) part[wave][lane >> (6 - LOG)] = sum[0];
  __syncthreads();
  if (threadIdx.x < VALUES) {
    const int row = threadIdx.x / kFeatures;
    const size_t feature = first + threadIdx.x % kFeatures;
    if (row < rows && feature < features) {
      double z = 0.0;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) z += part[k][threadIdx.x];
      const size_t at = (size_t)row * features + feature;
      if (bias) z += bias[feature];
      if (e.pre) e.pre[at] = z;
      double y = activate(e.activation, z);
      if (e.residual) y += e.residual[at];
      out[at] = y;
    }
  }
}

template <int ROWS, int DEPTH, int WAVES>
int launch_waves(hipStream_t s, const double* x, const double* w, const double* bias, double* out, const ActEpilogue& e,
                 int rows, size_t features, size_t length) {
  // a grid has fewer than 2^32 threads; more features take several launches, each of them long
  constexpr size_t kMostGroups = ((size_t)1 << 31) / (64 * WAVES);
  const size_t groups = (features + kFeatures - 1) / kFeatures;
  for (size_t g = 0; g < groups; g += kMostGroups) {
    const dim3 grid((unsigned)(groups - g < kMostGroups ? groups - g : kMostGroups));
    hipLaunchKernelGGL((linear_rows_kernel<ROWS, WAVES, DEPTH>), grid, dim3(64 * WAVES), 0, s, x, w, bias, out, e, rows,
                       features, length, g * kFeatures);
    RST_HIP(hipGetLastError());
  }
  return RST_OK;
}

template <int ROWS, int DEPTH>
int launch(hipStream_t s, const double* x, const double* w, const double* bias, double* out, const ActEpilogue& e,
           int rows, size_t features, size_t length) {
  // few weight rows: more wavefronts on each, so that the chip has loads enough in flight
  constexpr int MANY = ROWS == 8 ? 8 : 16;  // (sixteen leave 128 registers, and eight rows need more)
  if (features <= 1024) return launch_waves<ROWS, DEPTH, MANY>(s, x, w, bias, out, e, rows, features, length);
  return launch_waves<ROWS, DEPTH, 4>(s, x, w, bias, out, e, rows, features, length);
}

}  // namespace

bool linear_rows_supported(size_t rows, size_t features, size_t length) {
  if (length == 0) return false;  // (no product at all: the tiles write the bias)
  return rows <= 4 || (rows <= 8 && features * length >= (size_t)1 << 21);
}

int launch_linear_rows(hipStream_t s, const double* x, const double* w, const double* bias, double* out,
                       const ActEpilogue& e, size_t rows, size_t features, size_t length) {
  if (rows == 1) return launch<1, 4>(s, x, w, bias, out, e, (int)rows, features, length);
  if (rows == 2) return launch<2, 4>(s, x, w, bias, out, e, (int)rows, features, length);
  if (rows <= 4) return launch<4, 2>(s, x, w, bias, out, e, (int)rows, features, length);
  return launch<8, 1>(s, x, w, bias, out, e, (int)rows, features, length);
}

}  // namespace rst
