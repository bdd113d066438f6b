// Layer normalisation over each row, f64, forward and backward.
//
//   m = sum(x) / cols, v = sum((x - m)^2) / cols, r = 1 / sqrt(v + eps), y = (x - m) r * w + b
//   xh = (x - m) r, u = g * w:  dx = r (u - sum(u) / cols - xh sum(u xh) / cols) [+ residual]
//   dw = sum_rows(g xh) / rows, db = sum_rows(g) / rows
//
// Rows of up to a few thousand values stay in registers between the phases: the forward pass reads x
// once and takes the variance around the finished mean (no cancellation), the backward pass reads g
// and x once and keeps the two column sums of its rows in registers as well.  A workgroup of the
// backward pass walks over rows first, first + step, ... and leaves its column sums in the engine's
// scratch; a second launch adds them in workgroup order.  The grid is a function of the shape alone,
// so the order of every addition is too.
#include <climits>

#include "common.h"
#include "vec.h"

namespace rst {
namespace {

constexpr size_t kForwardCols = 16384;   // widest row the forward kernels keep in registers
constexpr size_t kBackwardCols = 8192;   // the backward kernels

// columns c, c + 1 of a row of `cols` values; 0 beyond the end
__device__ __forceinline__ v2u load_pair(const double* row, size_t c, size_t cols) {
  v2u v = {0.0, 0.0};
  if (c + 1 < cols) v = load2(row + c);
  else if (c < cols) v.x = row[c];
  return v;
}
__device__ __forceinline__ void store_pair(double* row, size_t c, size_t cols, v2u v) {
  if (c + 1 < cols) store2(row + c, v);
  else if (c < cols) row[c] = v.x;
}

// Sums of a and b over the TPR consecutive threads that share a row; every thread of the group gets the
// same bits.  scratch: 2 * TPR / 64 doubles (TPR > 64); a caller that reduces again before the next
// barrier passes another scratch.
template <int TPR>
__device__ __forceinline__ void group_sum2(double& a, double& b, double* scratch) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) {
    a += __shfl_xor(a, off);
    b += __shfl_xor(b, off);
  }
  if (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      scratch[2 * wave] = a;
      scratch[2 * wave + 1] = b;
    }
    __syncthreads();
    a = scratch[0];
    b = scratch[1];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      a += scratch[2 * w];
      b += scratch[2 * w + 1];
    }
  }
}

template <int TPR>
__device__ __forceinline__ double group_sum(double a, double* scratch) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) a += __shfl_xor(a, off);
  if (TPR > 64) {
    constexpr int NW = TPR / 64;
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = a;
    __syncthreads();
    a = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) a += scratch[w];
  }
  return a;
}

// ---- forward ------------------------------------------------------------------------------------
// TPR threads per row, IPT pairs per thread, BLOCK / TPR rows per workgroup.
template <int TPR, int IPT, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_forward_kernel(const double* x, const double* __restrict__ w,
                                                             const double* __restrict__ b, double* out, double* mean,
                                                             double* rstd, size_t rows, size_t cols, double eps) {
  static_assert(BLOCK % TPR == 0 && (TPR <= 64 || BLOCK == TPR), "unsupported shape");
  __shared__ double scratch[2][TPR > 64 ? TPR / 64 : 1];
  const int sub = threadIdx.x % TPR;
  const double n = (double)cols;
  // (one turn, unless there are more rows than a grid may have threads for; the turns are the same for
  // every thread of a workgroup that shares a row)
  const size_t step = (size_t)gridDim.x * (BLOCK / TPR);
  for (size_t row = (size_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR; row < rows; row += step) {
    const size_t base = row * cols;
    v2u v[IPT];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      v[i] = load_pair(x + base, 2 * (size_t)(sub + i * TPR), cols);
      sum += v[i].x + v[i].y;
    }
    const double m = group_sum<TPR>(sum, scratch[0]) / n;
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const size_t c = 2 * (size_t)(sub + i * TPR);
      v[i].x = c < cols ? v[i].x - m : 0.0;
      v[i].y = c + 1 < cols ? v[i].y - m : 0.0;
      sq = fma(v[i].x, v[i].x, sq);
      sq = fma(v[i].y, v[i].y, sq);
    }
    const double r = 1.0 / sqrt(group_sum<TPR>(sq, scratch[1]) / n + eps);
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const size_t c = 2 * (size_t)(sub + i * TPR);
      v2u y = v[i] * r;
      if (w) y *= load_pair(w, c, cols);
      if (b) y += load_pair(b, c, cols);
      store_pair(out + base, c, cols, y);
    }
    if (sub == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
  }
}

// Wider rows: one workgroup walks the row three times (mean, variance, result).
constexpr int kWideBlock = 1024;
__global__ __launch_bounds__(kWideBlock) void norm_forward_wide_kernel(const double* x, const double* __restrict__ w,
                                                                       const double* __restrict__ b, double* out,
                                                                       double* mean, double* rstd, size_t cols,
                                                                       double eps) {
  __shared__ double scratch[2][kWideBlock / 64];
  const size_t row = blockIdx.x;
  const double* src = x + row * cols;
  double sum = 0.0;
  for (size_t c = 2 * (size_t)threadIdx.x; c < cols; c += 2 * kWideBlock) {
    const v2u v = load_pair(src, c, cols);
    sum += v.x + v.y;
  }
  const double n = (double)cols;
  const double m = group_sum<kWideBlock>(sum, scratch[0]) / n;
  double sq = 0.0;
  for (size_t c = 2 * (size_t)threadIdx.x; c < cols; c += 2 * kWideBlock) {
    const v2u v = load_pair(src, c, cols);
    const double d0 = v.x - m, d1 = c + 1 < cols ? v.y - m : 0.0;
    sq = fma(d0, d0, sq);
    sq = fma(d1, d1, sq);
  }
  const double r = 1.0 / sqrt(group_sum<kWideBlock>(sq, scratch[1]) / n + eps);
  for (size_t c = 2 * (size_t)threadIdx.x; c < cols; c += 2 * kWideBlock) {
    v2u y = (load_pair(src, c, cols) - m) * r;
    if (w) y *= load_pair(w, c, cols);
    if (b) y += load_pair(b, c, cols);
    store_pair(out + row * cols, c, cols, y);
  }
  if (threadIdx.x == 0) {
    if (mean) mean[row] = m;
    if (rstd) rstd[row] = r;
  }
}

// ---- backward -----------------------------------------------------------------------------------
struct NormGrad {
  const double* grad;
  const double* x;
  const double* weight;    // NULL: ones
  const double* mean;
  const double* rstd;
  const double* residual;  // added to grad_input, or NULL
  double* grad_input;
  double* grad_weight;     // NULL: not wanted
  double* grad_bias;       // NULL: not wanted
  double* partial;         // [blocks][2][cols] column sums of the workgroups (more than one)
  size_t rows, cols;
};

template <int TPR, int IPT, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_backward_kernel(const NormGrad p) {
  static_assert(BLOCK % TPR == 0 && (TPR <= 64 || BLOCK == TPR), "unsupported shape");
  constexpr int RPB = BLOCK / TPR;  // rows at a time
  __shared__ double scratch[2][TPR > 64 ? 2 * TPR / 64 : 1];
  // the row groups' column sums meet here, four columns of a thread at a time
  __shared__ double meet[RPB > 1 ? 4 * BLOCK : 1];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const size_t cols = p.cols;
  const double n = (double)cols;
  v2u dw[IPT], db[IPT], w[IPT];
#pragma unroll
  for (int i = 0; i < IPT; ++i) {
    dw[i] = db[i] = (v2u){0.0, 0.0};
    w[i] = p.weight ? load_pair(p.weight, 2 * (size_t)(sub + i * TPR), cols) : (v2u){1.0, 1.0};
  }
  const size_t step = (size_t)gridDim.x * RPB;
  int turn = 0;
  // every thread of the workgroup makes the same number of turns (there is a barrier in each)
  for (size_t first = (size_t)blockIdx.x * RPB; first < p.rows; first += step, turn ^= 1) {
    const size_t row = first + group;
    const bool live = row < p.rows;
    const size_t base = (live ? row : 0) * cols, limit = live ? cols : 0;
    const double m = live ? p.mean[row] : 0.0, r = live ? p.rstd[row] : 0.0;
    v2u g[IPT], xh[IPT];
    double c1 = 0.0, c2 = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const size_t c = 2 * (size_t)(sub + i * TPR);
      g[i] = load_pair(p.grad + base, c, limit);
      xh[i] = load_pair(p.x + base, c, limit);
    }
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      // (beyond the row's end g is 0, and with it everything that is added)
      xh[i] = (xh[i] - m) * r;
      db[i] += g[i];
      dw[i] += g[i] * xh[i];
      g[i] *= w[i];
      c1 += g[i].x + g[i].y;
      c2 = fma(g[i].x, xh[i].x, c2);
      c2 = fma(g[i].y, xh[i].y, c2);
    }
    group_sum2<TPR>(c1, c2, scratch[turn]);
    c1 /= n;
    c2 /= n;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const size_t c = 2 * (size_t)(sub + i * TPR);
      v2u dx = (g[i] - c1 - xh[i] * c2) * r;
      if (p.residual) dx += load_pair(p.residual + base, c, limit);
      store_pair(p.grad_input + base, c, limit, dx);
    }
  }
  if (!p.grad_weight && !p.grad_bias) return;
  // the row groups' sums, added in group order
#pragma unroll
  for (int i = 0; i < IPT; ++i) {
    if (RPB > 1) {
      __syncthreads();
      meet[4 * threadIdx.x] = dw[i].x;
      meet[4 * threadIdx.x + 1] = dw[i].y;
      meet[4 * threadIdx.x + 2] = db[i].x;
      meet[4 * threadIdx.x + 3] = db[i].y;
      __syncthreads();
      if (group == 0) {
        for (int k = 1; k < RPB; ++k) {
          const double* other = meet + 4 * (k * TPR + sub);
          dw[i].x += other[0];
          dw[i].y += other[1];
          db[i].x += other[2];
          db[i].y += other[3];
        }
      }
    }
    if (group == 0) {
      const size_t c = 2 * (size_t)(sub + i * TPR);
      if (gridDim.x == 1) {
        const double rows = (double)p.rows;
        if (p.grad_weight) store_pair(p.grad_weight, c, cols, dw[i] / rows);
        if (p.grad_bias) store_pair(p.grad_bias, c, cols, db[i] / rows);
      } else {
        double* out = p.partial + (size_t)blockIdx.x * 2 * cols;
        store_pair(out, c, cols, dw[i]);
        store_pair(out + cols, c, cols, db[i]);
      }
    }
  }
}

// out[c] = (sum over the workgroups, in order, of partial[block][c]) / rows, c in [0, 2 cols): the
// weight's columns, then the bias's.  16 columns x 16 parts of the workgroups per launch workgroup; the
// parts are added in order.
__global__ __launch_bounds__(256) void norm_columns_kernel(const double* __restrict__ partial, double* grad_weight,
                                                           double* grad_bias, size_t cols, int blocks, double rows) {
  __shared__ double part[16][17];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  const size_t col = (size_t)blockIdx.x * 16 + c;
  double s = 0.0;
  if (col < 2 * cols)
    for (int i = k; i < blocks; i += 16) s += partial[(size_t)i * 2 * cols + col];
  part[k][c] = s;
  __syncthreads();
  if (k == 0 && col < 2 * cols) {
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += part[i][c];
    t /= rows;
    if (col < cols) {
      if (grad_weight) grad_weight[col] = t;
    } else if (grad_bias) {
      grad_bias[col - cols] = t;
    }
  }
}

// Wider rows: the two row sums first (a workgroup per row) ...
__global__ __launch_bounds__(kWideBlock) void norm_backward_rows_kernel(const NormGrad p, double* row_sums) {
  __shared__ double scratch[2 * kWideBlock / 64];
  const size_t row = blockIdx.x, cols = p.cols;
  const double m = p.mean[row], r = p.rstd[row];
  double c1 = 0.0, c2 = 0.0;
  for (size_t c = 2 * (size_t)threadIdx.x; c < cols; c += 2 * kWideBlock) {
    v2u g = load_pair(p.grad + row * cols, c, cols);
    const v2u xh = (load_pair(p.x + row * cols, c, cols) - m) * r;
    if (p.weight) g *= load_pair(p.weight, c, cols);
    c1 += g.x + g.y;
    c2 = fma(g.x, xh.x, c2);
    c2 = fma(g.y, xh.y, c2);
  }
  group_sum2<kWideBlock>(c1, c2, scratch);
  if (threadIdx.x == 0) {
    row_sums[2 * row] = c1 / (double)cols;
    row_sums[2 * row + 1] = c2 / (double)cols;
  }
}

// ... then strips of 512 columns by rows first, first + gridDim.y, ...: input gradient and column sums
__global__ __launch_bounds__(256) void norm_backward_strip_kernel(const NormGrad p, const double* __restrict__ row_sums) {
  const size_t cols = p.cols;
  const size_t c = (size_t)blockIdx.x * 512 + 2 * threadIdx.x;
  if (c >= cols) return;
  const v2u w = p.weight ? load_pair(p.weight, c, cols) : (v2u){1.0, 1.0};
  v2u dw = {0.0, 0.0}, db = {0.0, 0.0};
  for (size_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const v2u g = load_pair(p.grad + row * cols, c, cols);
    const double m = p.mean[row], r = p.rstd[row];
    const v2u xh = (load_pair(p.x + row * cols, c, cols) - m) * r;
    db += g;
    dw += g * xh;
    v2u dx = (g * w - row_sums[2 * row] - xh * row_sums[2 * row + 1]) * r;
    if (p.residual) dx += load_pair(p.residual + row * cols, c, cols);
    store_pair(p.grad_input + row * cols, c, cols, dx);
  }
  if (gridDim.y == 1) {
    const double rows = (double)p.rows;
    if (p.grad_weight) store_pair(p.grad_weight, c, cols, dw / rows);
    if (p.grad_bias) store_pair(p.grad_bias, c, cols, db / rows);
  } else {
    double* out = p.partial + (size_t)blockIdx.y * 2 * cols;
    store_pair(out, c, cols, dw);
    store_pair(out + cols, c, cols, db);
  }
}

// column sums of `blocks` workgroups -> the parameters' gradients
int finish_columns(hipStream_t s, const NormGrad& p, int blocks) {
  if (blocks <= 1 || (!p.grad_weight && !p.grad_bias)) return RST_OK;
  hipLaunchKernelGGL(norm_columns_kernel, dim3((unsigned)((2 * p.cols + 15) / 16)), dim3(256), 0, s, p.partial,
                     p.grad_weight, p.grad_bias, p.cols, blocks, (double)p.rows);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

template <int TPR, int IPT, int BLOCK>
int forward_rows(hipStream_t s, const double* x, const double* w, const double* b, double* out, double* mean,
                 double* rstd, size_t rows, size_t cols, double eps) {
  constexpr size_t RPB = BLOCK / TPR;
  constexpr size_t MAX_BLOCKS = ((size_t)1 << 31) / BLOCK;  // (a grid has fewer than 2^32 threads)
  size_t blocks = (rows + RPB - 1) / RPB;
  if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
  hipLaunchKernelGGL((norm_forward_kernel<TPR, IPT, BLOCK>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, x, w, b, out,
                     mean, rstd, rows, cols, eps);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

// MAX_BLOCKS: the workgroups that fit on the chip at once
template <int TPR, int IPT, int BLOCK, int MAX_BLOCKS>
int backward_rows(hipStream_t s, NormGrad p, double* workspace, size_t workspace_count) {
  constexpr size_t RPB = BLOCK / TPR;
  size_t blocks = (p.rows + RPB - 1) / RPB;
  if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
  if (blocks > 1 && blocks * 2 * p.cols > workspace_count)
    return fail(RST_ERR_UNSUPPORTED, "layer_norm_backward: the scratch holds %zu doubles", workspace_count);
  p.partial = workspace;
  hipLaunchKernelGGL((norm_backward_kernel<TPR, IPT, BLOCK>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, p);
  RST_HIP(hipGetLastError());
  return finish_columns(s, p, (int)blocks);
}

int backward_wide(hipStream_t s, NormGrad p, double* workspace, size_t workspace_count) {
  if (2 * p.rows > workspace_count)
    return fail(RST_ERR_UNSUPPORTED, "layer_norm_backward: %zu rows of %zu columns", p.rows, p.cols);
  p.partial = workspace + 2 * p.rows;
  const size_t strips = (p.cols + 511) / 512;
  size_t parts = (2048 + strips - 1) / strips;  // eight workgroups per CU
  if (parts > p.rows) parts = p.rows;
  const size_t room = (workspace_count - 2 * p.rows) / (2 * p.cols);
  if (parts > room) parts = room > 0 ? room : 1;
  hipLaunchKernelGGL(norm_backward_rows_kernel, dim3((unsigned)p.rows), dim3(kWideBlock), 0, s, p, workspace);
  RST_HIP(hipGetLastError());
  hipLaunchKernelGGL(norm_backward_strip_kernel, dim3((unsigned)strips, (unsigned)parts), dim3(256), 0, s, p,
                     workspace);
  RST_HIP(hipGetLastError());
  return finish_columns(s, p, (int)parts);
}

}  // namespace

int launch_layer_norm_forward(hipStream_t s, const double* x, const double* w, const double* b, double* out,
                              double* mean, double* rstd, size_t rows, size_t cols, double eps) {
  if (rows == 0 || cols == 0) return RST_OK;
  if (cols <= 16) return forward_rows<8, 1, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 64) return forward_rows<16, 2, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 128) return forward_rows<16, 4, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 256) return forward_rows<64, 2, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 512) return forward_rows<64, 4, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 1024) return forward_rows<64, 8, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 2048) return forward_rows<256, 4, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 4096) return forward_rows<256, 8, 256>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= 8192) return forward_rows<512, 8, 512>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  if (cols <= kForwardCols) return forward_rows<1024, 8, 1024>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  hipLaunchKernelGGL(norm_forward_wide_kernel, dim3((unsigned)rows), dim3(kWideBlock), 0, s, x, w, b, out, mean, rstd,
                     cols, eps);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

int launch_layer_norm_backward(hipStream_t s, const double* grad, const double* x, const double* weight,
                               const double* mean, const double* rstd, const double* residual, double* grad_input,
                               double* grad_weight, double* grad_bias, size_t rows, size_t cols, double* workspace,
                               size_t workspace_count) {
  if (rows == 0 || cols == 0) return RST_OK;
  const NormGrad p{grad, x, weight, mean, rstd, residual, grad_input, grad_weight, grad_bias, nullptr, rows, cols};
  if (cols <= 16) return backward_rows<8, 1, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 64) return backward_rows<16, 2, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 128) return backward_rows<16, 4, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 256) return backward_rows<64, 2, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 512) return backward_rows<64, 4, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 1024) return backward_rows<128, 4, 128, 1024>(s, p, workspace, workspace_count);
  if (cols <= 2048) return backward_rows<256, 4, 256, 1024>(s, p, workspace, workspace_count);
  if (cols <= 4096) return backward_rows<512, 4, 512, 512>(s, p, workspace, workspace_count);
  if (cols <= kBackwardCols) return backward_rows<1024, 4, 1024, 256>(s, p, workspace, workspace_count);
  return backward_wide(s, p, workspace, workspace_count);
}

}  // namespace rst
