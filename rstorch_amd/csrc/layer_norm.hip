// Layer normalisation over each row, f64, forward and backward.
//
//   m = sum(x) / cols, v = sum((x - m)^2) / cols, r = 1 / sqrt(v + eps), y = (x - m) r * w + b
//   xh = (x - m) r, u = g * w:  dx = r (u - sum(u) / cols - xh sum(u xh) / cols) [+ residual]
//   dw = sum_rows(g xh) / rows, db = sum_rows(g) / rows
//
// Both are bound by HBM: 16 bytes an element forward, 24 backward (32 with the residual).  Rows of up to a
// few thousand values stay in registers between the phases: the forward pass reads x once and takes the
// variance around the finished mean (no cancellation), the backward pass reads g and x once and keeps the
// two column sums of its rows in registers as well.  A workgroup walks over rows first, first + step, ...
// with the parameters in registers and the loads of the next row issued before this one is worked on, so
// that the trip to memory and the two reductions of a row overlap.  The backward pass leaves its column sums in the
// engine's scratch and a second launch adds them in workgroup order; a batch that one workgroup handles in a
// few turns needs no second launch.  The grid is a function of the shape alone, so the order of every
// addition is too.
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

// A thread's share of a row that TPR consecutive threads hold: IPT pairs, pair i at column
// 2 (sub + i TPR), with 2 TPR (IPT - 1) < cols <= 2 TPR IPT: only the last pair may reach beyond the row's end
// (FULL: not even that).  Such a pair is loaded from the row's last two columns (there are two at least), so
// that no load is behind a branch, and what does not belong to it is zeroed when it is used.
template <int TPR, int IPT, bool FULL>
struct Span {
  int sub;
  bool has_first, has_both;  // of the last pair
  uint32_t last;             // byte offset of its load
  __device__ __forceinline__ Span(int s, int cols) : sub(s) {
    const int c = 2 * (sub + (IPT - 1) * TPR);
    has_first = FULL || c < cols;
    has_both = FULL || c + 1 < cols;
    last = 8u * (uint32_t)(has_both ? c : cols - 2);
  }
  __device__ __forceinline__ bool ragged(int i) const { return !FULL && i == IPT - 1; }
  __device__ __forceinline__ bool first(int i) const { return !ragged(i) || has_first; }
  __device__ __forceinline__ bool both(int i) const { return !ragged(i) || has_both; }
  __device__ __forceinline__ const double* place(const double* row, int i) const {
    const uint32_t at = ragged(i) ? last : 16u * (uint32_t)(sub + i * TPR);
    return reinterpret_cast<const double*>(reinterpret_cast<const char*>(row) + at);
  }
  __device__ __forceinline__ void load(v2u* v, const double* row) const {
#pragma unroll
    for (int i = 0; i < IPT; ++i) v[i] = load2_stream(place(row, i));
  }
  // a parameter row (read again by every workgroup); NULL: `value` everywhere
  __device__ __forceinline__ v2u parameter(int i, const double* row, double value) const {
    if (!row) return (v2u){value, value};
    return settle(i, load2(place(row, i)));
  }
  __device__ __forceinline__ void parameter(v2u* v, const double* row, double value) const {
#pragma unroll
    for (int i = 0; i < IPT; ++i) v[i] = parameter(i, row, value);
  }
  // the pair as it is in the row, 0 beyond the end
  __device__ __forceinline__ v2u settle(int i, v2u v) const {
    if (ragged(i)) {
      v.x = has_both ? v.x : has_first ? v.y : 0.0;
      v.y = has_both ? v.y : 0.0;
    }
    return v;
  }
  __device__ __forceinline__ void store(double* row, int i, v2u v) const {
    double* to = row + 2 * (sub + i * TPR);
    if (both(i)) store2(to, v);
    else if (first(i)) to[0] = v.x;
  }
};

// Sums of a and b over the TPR consecutive threads that share a row; every thread of the group gets the
// same bits.  scratch: the group's 2 * TPR / 64 doubles (TPR > 64); a caller that reduces again before the
// next barrier passes others.
template <int TPR>
__device__ __forceinline__ void group_sum2(double& a, double& b, double* scratch) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) {
    a += __shfl_xor(a, off);
    b += __shfl_xor(b, off);
  }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = (threadIdx.x % TPR) >> 6;
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
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    if ((threadIdx.x & 63) == 0) scratch[(threadIdx.x % TPR) >> 6] = a;
    __syncthreads();
    a = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) a += scratch[w];
  }
  return a;
}

// the row a thread group works on, in scalar registers where it is the same for the whole wavefront
template <int TPR>
__device__ __forceinline__ int group_of_thread() {
  const int g = (int)threadIdx.x / TPR;
  return TPR >= 64 ? __builtin_amdgcn_readfirstlane(g) : g;
}

// ---- forward ------------------------------------------------------------------------------------
// TPR threads per row, IPT pairs per thread, BLOCK / TPR rows per workgroup and turn.  AHEAD: the next row's loads
// are issued before this row is worked on; HOLD: the parameters stay in registers; WAVES per SIMD to leave registers for.
// Bound by HBM, a row is read once: 16384 x 4096 197 us (5.5 TB/s; copies of whole rows in this pattern reach 5.7 to 6.1),
// 2047 x 1023 9.2 us (3.6 TB/s, cache and HBM).
template <int TPR, int IPT, int BLOCK, bool FULL, bool AHEAD, bool HOLD, int WAVES>
__global__ __launch_bounds__(BLOCK, WAVES) void norm_forward_kernel(const double* x, const double* w, const double* b,
                                                             double* out, double* mean, double* rstd, int rows,
                                                             int cols, double eps) {
  static_assert(BLOCK % TPR == 0 && (TPR <= 64 || BLOCK == TPR), "unsupported shape");
  __shared__ double scratch[2][TPR > 64 ? TPR / 64 : 1];
  const Span<TPR, IPT, FULL> span((int)threadIdx.x % TPR, cols);
  const double n = (double)cols;
  const int step = (int)gridDim.x * (BLOCK / TPR);
  int row = (int)blockIdx.x * (BLOCK / TPR) + group_of_thread<TPR>();
  if (row >= rows) return;  // (a whole workgroup, or a group that meets no barrier)
  v2u v[IPT], next[IPT], wv[IPT], bv[IPT];
  span.load(v, x + (size_t)row * cols);
  if (HOLD) {
    span.parameter(wv, w, 1.0);
    span.parameter(bv, b, 0.0);
  }
  for (;;) {
    const bool more = row < rows - step;
    if (AHEAD && more) span.load(next, x + (size_t)(row + step) * cols);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      v[i] = span.settle(i, v[i]);
      sum += v[i].x + v[i].y;
    }
    const double m = group_sum<TPR>(sum, scratch[0]) / n;
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      v[i].x = span.first(i) ? v[i].x - m : 0.0;
      v[i].y = span.both(i) ? v[i].y - m : 0.0;
      sq = fma(v[i].x, v[i].x, sq);
      sq = fma(v[i].y, v[i].y, sq);
    }
    const double r = 1.0 / sqrt(group_sum<TPR>(sq, scratch[1]) / n + eps);
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const v2u wi = HOLD ? wv[i] : span.parameter(i, w, 1.0), bi = HOLD ? bv[i] : span.parameter(i, b, 0.0);
      span.store(out + (size_t)row * cols, i, v[i] * r * wi + bi);
      if (!HOLD) __builtin_amdgcn_sched_barrier(0);  // (all parameters at once would not fit the registers)
    }
    if (span.sub == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    if (!more) break;
    row += step;
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < IPT; ++i) v[i] = next[i];
    } else {
      span.load(v, x + (size_t)row * cols);
    }
  }
}

// Rows too wide for the registers, and rows of one value (no pair to load): one workgroup walks the row twice.  The
// first walk takes mean and squared deviations together: a thread's batch of sixteen values gets its own mean and
// deviations in registers (no cancellation), which join the thread's running ones; the threads' means then give the
// row's, and the deviations are moved onto it: sum_i (S_i + n_i (m_i - m)^2).  All of this is done on x minus the row's
// first value, which is within sqrt(cols) standard deviations of the mean: a rounding of the means is then small
// against the deviations also where the values have a large common part.  1024 x 32768: 171 us (184 in three
// walks; 207 with the row kept half in registers and half in LDS, which leaves one workgroup per CU and nothing to overlap
// its phases with).
template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_forward_wide_kernel(const double* x, const double* __restrict__ w,
                                                                  const double* __restrict__ b, double* out,
                                                                  double* mean, double* rstd, size_t rows, size_t cols,
                                                                  double eps) {
  __shared__ double scratch[2][BLOCK / 64];
  constexpr size_t STEP = 2 * BLOCK;
  constexpr int DEPTH = 8;
  const double n = (double)cols;
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const double* src = x + row * cols;
    const double shift = src[0];
    double count = 0.0, centre = 0.0, spread = 0.0;  // of what this thread has read
    // joins `values` more values of the given mean and squared deviations
    auto join = [&](double values, double m, double s) {
      const double total = count + values, delta = m - centre;
      const double share = values / total;
      centre = fma(delta, share, centre);
      spread += fma(delta * delta, count * share, s);
      count = total;
    };
    size_t c = 2 * (size_t)threadIdx.x;
    for (; c + (DEPTH - 1) * STEP + 1 < cols; c += DEPTH * STEP) {
      v2u t[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) t[d] = load2(src + c + d * STEP);
      double sum = 0.0, sq = 0.0;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        t[d] -= shift;
        sum += t[d].x + t[d].y;
      }
      const double m = sum * (0.5 / DEPTH);
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        sq = fma(t[d].x - m, t[d].x - m, sq);
        sq = fma(t[d].y - m, t[d].y - m, sq);
      }
      join(2.0 * DEPTH, m, sq);
    }
    for (; c < cols; c += STEP) {
      const v2u t = load_pair(src, c, cols) - shift;
      if (c + 1 < cols) {
        const double half = 0.5 * (t.x - t.y);
        join(2.0, t.y + half, 2.0 * half * half);
      } else {
        join(1.0, t.x, 0.0);
      }
    }
    const double moved = group_sum<BLOCK>(count * centre, scratch[0]) / n;
    const double m = shift + moved, off = centre - moved;
    const double r = 1.0 / sqrt(group_sum<BLOCK>(fma(count * off, off, spread), scratch[1]) / n + eps);
    c = 2 * (size_t)threadIdx.x;
    auto finish = [&](v2u v, size_t at) {
      v2u y = (v - m) * r;
      if (w) y *= load_pair(w, at, cols);
      if (b) y += load_pair(b, at, cols);
      store_pair(out + row * cols, at, cols, y);
    };
    for (; c + 3 * STEP + 1 < cols; c += 4 * STEP) {
      v2u t[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) t[d] = load2(src + c + d * STEP);
#pragma unroll
      for (int d = 0; d < 4; ++d) finish(t[d], c + d * STEP);
    }
    for (; c < cols; c += STEP) finish(load_pair(src, c, cols), c);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    __syncthreads();  // (a wavefront without columns would run ahead into the next row's scratch)
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
  int rows, cols;
};

// A row of grad and x is read once, into registers: the two sums of a row (of u and of u xh) join across its threads, then
// grad_input is written and the thread's columns of the parameters' gradients, which a workgroup keeps in registers over
// all its rows, move on.  Bound by HBM: 8192 x 4096 with a residual 200 us (5.4 TB/s), 2047 x 1023 14.5 us (3.5 TB/s: eight
// rows a workgroup, and the sums' way out is as long as two of them).
template <int TPR, int IPT, int BLOCK, bool FULL, bool AHEAD, bool HOLD, int WAVES>
__global__ __launch_bounds__(BLOCK, WAVES) void norm_backward_kernel(const NormGrad p) {
  static_assert(BLOCK % TPR == 0, "whole rows per workgroup");
  constexpr int RPB = BLOCK / TPR;  // rows at a time
  __shared__ double scratch[2][RPB][TPR > 64 ? 2 * TPR / 64 : 1];
  // the row groups' column sums meet here, four columns of a thread at a time
  __shared__ double meet[RPB > 1 ? 4 * BLOCK : 1];
  const int group = group_of_thread<TPR>();
  const Span<TPR, IPT, FULL> span((int)threadIdx.x % TPR, p.cols);
  const double n = (double)p.cols;
  v2u dw[IPT], db[IPT], w[IPT];
  const int step = (int)gridDim.x * RPB;
  // Every thread of the workgroup makes the same number of turns (there may be a barrier in each); a group
  // whose row does not exist works on the last row with a gradient of zero and stores nothing.
  int first = (int)blockIdx.x * RPB;
  v2u g[IPT], x[IPT], next_g[IPT], next_x[IPT];
  double m = 0.0, r = 0.0, next_m = 0.0, next_r = 0.0;
  auto fetch = [&](int row, v2u* gv, v2u* xv, double& mv, double& rv) {
    const int at = row < p.rows ? row : p.rows - 1;
    span.load(gv, p.grad + (size_t)at * p.cols);
    span.load(xv, p.x + (size_t)at * p.cols);
    mv = p.mean[at];
    rv = p.rstd[at];
  };
  fetch(first + group, g, x, m, r);
  if (HOLD) span.parameter(w, p.weight, 1.0);
#pragma unroll
  for (int i = 0; i < IPT; ++i) dw[i] = db[i] = (v2u){0.0, 0.0};
  int turn = 0;
  for (;;) {
    const int row = first + group;
    const bool live = row < p.rows;
    const bool more = first < p.rows - step;
    if (AHEAD && more) fetch(row + step, next_g, next_x, next_m, next_r);
    v2u res[IPT];
    if (HOLD && p.residual) span.load(res, p.residual + (size_t)(live ? row : p.rows - 1) * p.cols);
    double c1 = 0.0, c2 = 0.0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      // (beyond the row's end, and without a row, g is 0 and with it everything that is added: the
      // products are selected, not multiplied, since x may be infinite there)
      g[i] = span.settle(i, g[i]);
      x[i] = (span.settle(i, x[i]) - m) * r;
      v2u gx = g[i] * x[i];
      gx.x = span.first(i) ? gx.x : 0.0;
      gx.y = span.both(i) ? gx.y : 0.0;
      if (RPB > 1) {
        gx = live ? gx : (v2u){0.0, 0.0};
        g[i] = live ? g[i] : (v2u){0.0, 0.0};
      }
      db[i] += g[i];
      dw[i] += gx;
      const v2u wi = HOLD ? w[i] : span.parameter(i, p.weight, 1.0);
      g[i] *= wi;
      c1 += g[i].x + g[i].y;
      c2 = fma(gx.x, wi.x, c2);
      c2 = fma(gx.y, wi.y, c2);
    }
    group_sum2<TPR>(c1, c2, scratch[turn][group]);
    c1 /= n;
    c2 /= n;
    if (live) {
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        v2u dx = (g[i] - c1 - x[i] * c2) * r;
        if (p.residual) dx += HOLD ? span.settle(i, res[i]) : span.parameter(i, p.residual + (size_t)row * p.cols, 0.0);
        span.store(p.grad_input + (size_t)row * p.cols, i, dx);
      }
    }
    if (!more) break;
    first += step;
    turn ^= 1;
    if (AHEAD) {
      m = next_m;
      r = next_r;
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        g[i] = next_g[i];
        x[i] = next_x[i];
      }
    } else {
      fetch(first + group, g, x, m, r);
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
          const double* other = meet + 4 * (k * TPR + span.sub);
          dw[i].x += other[0];
          dw[i].y += other[1];
          db[i].x += other[2];
          db[i].y += other[3];
        }
      }
    }
    if (group == 0) {
      if (gridDim.x == 1) {
        const double rows = (double)p.rows;
        if (p.grad_weight) span.store(p.grad_weight, i, dw[i] / rows);
        if (p.grad_bias) span.store(p.grad_bias, i, db[i] / rows);
      } else {
        double* out = p.partial + (size_t)blockIdx.x * 2 * p.cols;
        span.store(out, i, dw[i]);
        span.store(out + p.cols, i, db[i]);
      }
    }
  }
}

// out[c] = (sum over the workgroups, in order, of partial[block][c]) / rows, c in [0, 2 cols): the
// weight's columns, then the bias's.  5 us behind 8192 x 4096 (256 sets of 8192 sums).  16 columns x 16 parts of the
// workgroups per launch workgroup; the parts are added in order.
__global__ __launch_bounds__(256) void norm_columns_kernel(const double* __restrict__ partial, double* grad_weight,
                                                           double* grad_bias, size_t cols, int blocks, double rows) {
  __shared__ double part[16][17];
  const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
  const size_t col = (size_t)blockIdx.x * 16 + c;
  double s = 0.0;
  if (col < 2 * cols) {
    int i = k;
    for (; i + 7 * 16 < blocks; i += 8 * 16) {
      double t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = partial[(size_t)(i + 16 * j) * 2 * cols + col];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += t[j];
    }
    for (; i < blocks; i += 16) s += partial[(size_t)i * 2 * cols + col];
  }
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

// Wider rows, and rows of one value: the two row sums first (a workgroup per row; 1065 x 15566 58 us, 4.6 TB/s) ...
template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_backward_rows_kernel(const NormGrad p, double* row_sums) {
  __shared__ double scratch[2 * BLOCK / 64];
  const size_t cols = p.cols;
  for (size_t row = blockIdx.x; row < (size_t)p.rows; row += gridDim.x) {
    const double m = p.mean[row], r = p.rstd[row];
    double c1 = 0.0, c2 = 0.0;
    for (size_t c = 2 * (size_t)threadIdx.x; c < cols; c += 2 * BLOCK) {
      v2u g = load_pair(p.grad + row * cols, c, cols);
      v2u xh = (load_pair(p.x + row * cols, c, cols) - m) * r;
      if (c + 1 >= cols) xh.y = 0.0;
      if (p.weight) g *= load_pair(p.weight, c, cols);
      c1 += g.x + g.y;
      c2 = fma(g.x, xh.x, c2);
      c2 = fma(g.y, xh.y, c2);
    }
    group_sum2<BLOCK>(c1, c2, scratch);
    if (threadIdx.x == 0) {
      row_sums[2 * row] = c1 / (double)cols;
      row_sums[2 * row + 1] = c2 / (double)cols;
    }
    __syncthreads();
  }
}

// ... then strips of 512 columns by rows first, first + gridDim.y, ...: input gradient and column sums (69 us, 5.8 TB/s)
__global__ __launch_bounds__(256) void norm_backward_strip_kernel(const NormGrad p, const double* __restrict__ row_sums) {
  const size_t cols = p.cols;
  const size_t c = (size_t)blockIdx.x * 512 + 2 * threadIdx.x;
  if (c >= cols) return;
  const v2u w = p.weight ? load_pair(p.weight, c, cols) : (v2u){1.0, 1.0};
  v2u dw = {0.0, 0.0}, db = {0.0, 0.0};
  for (size_t row = blockIdx.y; row < (size_t)p.rows; row += gridDim.y) {
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
  hipLaunchKernelGGL(norm_columns_kernel, dim3((unsigned)((2 * (size_t)p.cols + 15) / 16)), dim3(256), 0, s, p.partial,
                     p.grad_weight, p.grad_bias, (size_t)p.cols, blocks, (double)p.rows);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

// MAX_BLOCKS: the workgroups that fit on the chip at once, about
template <int TPR, int IPT, int BLOCK, int MAX_BLOCKS, bool AHEAD = true, bool HOLD = true, int WAVES = 1>
int forward_rows(hipStream_t s, const double* x, const double* w, const double* b, double* out, double* mean,
                 double* rstd, size_t rows, size_t cols, double eps) {
  constexpr size_t RPB = BLOCK / TPR;
  size_t blocks = (rows + RPB - 1) / RPB;
  if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
  if (cols == 2 * TPR * IPT)
    hipLaunchKernelGGL((norm_forward_kernel<TPR, IPT, BLOCK, true, AHEAD, HOLD, WAVES>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, x, w,
                       b, out, mean, rstd, (int)rows, (int)cols, eps);
  else
    hipLaunchKernelGGL((norm_forward_kernel<TPR, IPT, BLOCK, false, AHEAD, HOLD, WAVES>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, x, w,
                       b, out, mean, rstd, (int)rows, (int)cols, eps);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

template <int BLOCK>
int forward_wide(hipStream_t s, const double* x, const double* w, const double* b, double* out, double* mean,
                 double* rstd, size_t rows, size_t cols, double eps) {
  const size_t most = ((size_t)1 << 31) / BLOCK;  // (a grid has fewer than 2^32 threads)
  hipLaunchKernelGGL((norm_forward_wide_kernel<BLOCK>), dim3((unsigned)(rows < most ? rows : most)),
                     dim3(BLOCK), 0, s, x, w, b, out, mean, rstd, rows, cols, eps);
  RST_HIP(hipGetLastError());
  return RST_OK;
}

template <int TPR, int IPT, int BLOCK, int MAX_BLOCKS, bool AHEAD = true, bool HOLD = true, int WAVES = 1>
int backward_rows(hipStream_t s, NormGrad p, double* workspace, size_t workspace_count) {
  constexpr size_t RPB = BLOCK / TPR;
  size_t blocks = ((size_t)p.rows + RPB - 1) / RPB;
  // a handful of turns of one workgroup are over before a second launch would have begun
  if (blocks <= 4) blocks = 1;
  if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
  if (blocks > 1 && blocks * 2 * p.cols > workspace_count)
    return fail(RST_ERR_UNSUPPORTED, "layer_norm_backward: the scratch holds %zu doubles", workspace_count);
  p.partial = workspace;
  if (p.cols == 2 * TPR * IPT)
    hipLaunchKernelGGL((norm_backward_kernel<TPR, IPT, BLOCK, true, AHEAD, HOLD, WAVES>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, p);
  else
    hipLaunchKernelGGL((norm_backward_kernel<TPR, IPT, BLOCK, false, AHEAD, HOLD, WAVES>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, p);
  RST_HIP(hipGetLastError());
  return finish_columns(s, p, (int)blocks);
}

template <int BLOCK>
int backward_wide(hipStream_t s, NormGrad p, double* workspace, size_t workspace_count) {
  const size_t rows = p.rows, cols = p.cols;
  if (2 * rows > workspace_count) return fail(RST_ERR_UNSUPPORTED, "layer_norm_backward: %zu rows of %zu columns", rows, cols);
  p.partial = workspace + 2 * rows;
  const size_t strips = (cols + 511) / 512;
  size_t parts = (2048 + strips - 1) / strips;  // eight workgroups per CU
  if (parts > rows) parts = rows;
  const size_t room = (workspace_count - 2 * rows) / (2 * cols);
  if (parts > room) parts = room > 0 ? room : 1;
  const size_t most = ((size_t)1 << 31) / BLOCK;
  hipLaunchKernelGGL(norm_backward_rows_kernel<BLOCK>, dim3((unsigned)(rows < most ? rows : most)), dim3(BLOCK), 0, s,
                     p, workspace);
  RST_HIP(hipGetLastError());
  hipLaunchKernelGGL(norm_backward_strip_kernel, dim3((unsigned)strips, (unsigned)parts), dim3(256), 0, s, p,
                     workspace);
  RST_HIP(hipGetLastError());
  return finish_columns(s, p, (int)parts);
}

// the fewest pairs per thread, IPT to MOST, that hold the row
template <int TPR, int IPT, int MOST, int BLOCK, int MAX_BLOCKS, bool AHEAD, bool HOLD, int WAVES>
int forward_pick(hipStream_t s, const double* x, const double* w, const double* b, double* out, double* mean,
                 double* rstd, size_t rows, size_t cols, double eps) {
  if constexpr (IPT < MOST) {
    if (cols > 2 * TPR * IPT)
      return forward_pick<TPR, IPT + 1, MOST, BLOCK, MAX_BLOCKS, AHEAD, HOLD, WAVES>(s, x, w, b, out, mean, rstd, rows, cols, eps);
  }
  return forward_rows<TPR, IPT, BLOCK, MAX_BLOCKS, AHEAD, HOLD, WAVES>(s, x, w, b, out, mean, rstd, rows, cols, eps);
}

template <int TPR, int IPT, int MOST, int BLOCK, int MAX_BLOCKS, bool AHEAD, bool HOLD>
int backward_pick(hipStream_t s, const NormGrad& p, double* workspace, size_t workspace_count) {
  if constexpr (IPT < MOST) {
    if (p.cols > 2 * TPR * IPT)
      return backward_pick<TPR, IPT + 1, MOST, BLOCK, MAX_BLOCKS, AHEAD, HOLD>(s, p, workspace, workspace_count);
  }
  return backward_rows<TPR, IPT, BLOCK, MAX_BLOCKS, AHEAD, HOLD>(s, p, workspace, workspace_count);
}

}  // namespace

int launch_layer_norm_forward(hipStream_t s, const double* x, const double* w, const double* b, double* out,
                              double* mean, double* rstd, size_t rows, size_t cols, double eps) {
  if (rows == 0 || cols == 0) return RST_OK;
  // Up to 1024 columns a workgroup takes its rows and ends: enough workgroups fit on a CU to overlap their trips to
  // memory (2047 x 1023: 9.2 us, 11 with the loads of a next row held in registers); above, workgroups stay and load
  // ahead (8192 x 4096: 96 us, 110 one row at a time).
  constexpr int ALL = 1 << 22;  // (a grid has fewer than 2^32 threads)
#define RST_NORM_ARGS s, x, w, b, out, mean, rstd, rows, cols, eps
  if (cols == 1) return forward_wide<64>(RST_NORM_ARGS);
  if (cols <= 16) return forward_pick<8, 1, 1, 256, ALL, false, true, 1>(RST_NORM_ARGS);
  if (cols <= 64) return forward_pick<16, 1, 2, 256, ALL, false, true, 1>(RST_NORM_ARGS);
  if (cols <= 128) return forward_pick<32, 2, 2, 256, ALL, false, true, 1>(RST_NORM_ARGS);
  if (cols <= 512) return forward_pick<64, 2, 4, 256, ALL, false, true, 4>(RST_NORM_ARGS);
  if (cols <= 1024) return forward_pick<128, 3, 4, 128, ALL, false, true, 4>(RST_NORM_ARGS);
  if (cols <= 2048) return forward_pick<256, 3, 4, 256, 1280, true, true, 4>(RST_NORM_ARGS);
  if (cols <= 4096) return forward_pick<256, 5, 8, 256, 512, true, true, 2>(RST_NORM_ARGS);
  if (cols <= 8192) return forward_pick<512, 5, 8, 512, 256, true, true, 2>(RST_NORM_ARGS);
  if (cols <= kForwardCols) return forward_pick<1024, 5, 8, 1024, 256, false, false, 4>(RST_NORM_ARGS);
  return forward_wide<1024>(RST_NORM_ARGS);
#undef RST_NORM_ARGS
}

int launch_layer_norm_backward(hipStream_t s, const double* grad, const double* x, const double* weight,
                               const double* mean, const double* rstd, const double* residual, double* grad_input,
                               double* grad_weight, double* grad_bias, size_t rows, size_t cols, double* workspace,
                               size_t workspace_count) {
  if (rows == 0 || cols == 0) return RST_OK;
  const NormGrad p{grad, x, weight, mean, rstd, residual, grad_input, grad_weight, grad_bias, nullptr, (int)rows, (int)cols};
  // Workgroups stay for many rows, so that few sets of column sums are written and added up again.
  if (cols == 1) return backward_wide<64>(s, p, workspace, workspace_count);
  if (cols <= 16) return backward_pick<8, 1, 1, 256, 512, true, true>(s, p, workspace, workspace_count);
  if (cols <= 64) return backward_pick<16, 1, 2, 256, 512, true, true>(s, p, workspace, workspace_count);
  if (cols <= 128) return backward_pick<32, 2, 2, 512, 256, true, true>(s, p, workspace, workspace_count);
  if (cols <= 512) return backward_pick<64, 2, 4, 512, 256, true, true>(s, p, workspace, workspace_count);
  if (cols <= 1024) return backward_pick<128, 3, 4, 512, 256, true, true>(s, p, workspace, workspace_count);
  if (cols <= 2048) return backward_pick<256, 3, 4, 512, 256, true, true>(s, p, workspace, workspace_count);
  if (cols <= 4096) return backward_pick<512, 3, 4, 512, 256, true, true>(s, p, workspace, workspace_count);
  if (cols <= kBackwardCols) return backward_pick<512, 5, 8, 512, 256, false, false>(s, p, workspace, workspace_count);
  return backward_wide<1024>(s, p, workspace, workspace_count);
}

}  // namespace rst
