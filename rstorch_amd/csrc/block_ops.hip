// Operator-level C ABI of the residual block: layer norm, dropout, activations and the Linear layer
// with activation and residual.  Argument checking and dispatch; the reference has no counterpart, the
// conventions (division by the batch, gradients overwritten) are those of src/module/linear.rs:43-69.
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "common.h"

using namespace rst;

namespace {

int check_dim(const char* who, size_t v, const char* what) {
  if (v > kMostExtent) return fail(RST_ERR_UNSUPPORTED, "%s: %s = %zu exceeds 2^31-128", who, what, v);
  return RST_OK;
}

int check_activation(const char* who, int activation) {
  if (activation < RST_ACT_NONE || activation > RST_ACT_SILU)
    return fail(RST_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", who, activation);
  return RST_OK;
}

int check_probability(const char* who, double p) {
  if (!(p >= 0.0 && p < 1.0)) return fail(RST_ERR_INVALID_ARGUMENT, "%s: p = %g is not in [0, 1)", who, p);
  return RST_OK;
}

// An array of an entry point; count 0: not read or written in this call.
struct Range {
  const double* first;
  size_t count;
};
bool overlap(const Range& a, const Range& b) {
  if (!a.first || !b.first || a.count == 0 || b.count == 0) return false;
  // (in doubles: a byte count of the largest extents does not fit)
  const uintptr_t i = reinterpret_cast<uintptr_t>(a.first) / 8, j = reinterpret_cast<uintptr_t>(b.first) / 8;
  return i < j + b.count && j < i + a.count;
}
// An output over something that workgroups still read or write while it is written.
bool overlap_any(const Range& out, std::initializer_list<Range> others) {
  for (const Range& other : others)
    if (overlap(out, other)) return true;
  return false;
}
// ... over an array that each element is read from just before it is written to: that array itself is fine
bool overlap_shifted(const Range& out, const Range& in) { return out.first != in.first && overlap(out, in); }

}  // namespace

extern "C" {

int rst_layer_norm_forward(rst_engine* e, const double* x, const double* weight, const double* bias, double* out,
                           double* mean, double* rstd, size_t rows, size_t cols, double eps) {
  RST_TRY(engine_activate(e));
  if (!(eps >= 0.0 && std::isfinite(eps)))
    return fail(RST_ERR_INVALID_ARGUMENT, "layer_norm_forward: eps = %g", eps);
  if (rows == 0) return RST_OK;
  if (cols == 0) return fail(RST_ERR_SHAPE, "layer_norm_forward: rows without columns have no mean");
  if (!x || !out) return fail(RST_ERR_INVALID_ARGUMENT, "layer_norm_forward: null operand");
  RST_TRY(check_dim("layer_norm_forward", rows, "rows"));
  RST_TRY(check_dim("layer_norm_forward", cols, "cols"));
  return launch_layer_norm_forward(e->stream, x, weight, bias, out, mean, rstd, rows, cols, eps);
}

int rst_layer_norm_backward(rst_engine* e, const double* grad, const double* x, const double* weight,
                            const double* mean, const double* rstd, const double* residual_grad, double* grad_input,
                            double* grad_weight, double* grad_bias, size_t rows, size_t cols) {
  RST_TRY(engine_activate(e));
  if (rows == 0 || cols == 0) return fail(RST_ERR_SHAPE, "layer_norm_backward of a %zu x %zu array", rows, cols);
  if (!grad || !x || !mean || !rstd || !grad_input)
    return fail(RST_ERR_INVALID_ARGUMENT, "layer_norm_backward: null operand");
  RST_TRY(check_dim("layer_norm_backward", rows, "rows"));
  RST_TRY(check_dim("layer_norm_backward", cols, "cols"));
  return launch_layer_norm_backward(e->stream, grad, x, weight, mean, rstd, residual_grad, grad_input, grad_weight,
                                    grad_bias, rows, cols, e->d_gemm_ws, e->gemm_ws_count);
}

int rst_dropout_forward(rst_engine* e, const double* x, const double* residual, double* out, size_t count, double p,
                        uint64_t seed, uint64_t stream) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_probability("dropout_forward", p));
  if (count && (!x || !out)) return fail(RST_ERR_INVALID_ARGUMENT, "dropout_forward: null operand");
  return launch_dropout(e->stream, x, residual, out, count, p, seed, stream);
}

int rst_dropout_backward(rst_engine* e, const double* grad, double* out, size_t count, double p, uint64_t seed,
                         uint64_t stream) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_probability("dropout_backward", p));
  if (count && (!grad || !out)) return fail(RST_ERR_INVALID_ARGUMENT, "dropout_backward: null operand");
  return launch_dropout(e->stream, grad, nullptr, out, count, p, seed, stream);
}

int rst_activation_forward(rst_engine* e, const double* x, const double* residual, double* out, size_t count,
                           int activation) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_activation("activation_forward", activation));
  if (count && (!x || !out)) return fail(RST_ERR_INVALID_ARGUMENT, "activation_forward: null operand");
  return launch_act_forward(e->stream, activation, x, residual, out, count);
}

int rst_activation_backward(rst_engine* e, const double* grad, const double* pre, const double* residual, double* out,
                            size_t count, int activation) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_activation("activation_backward", activation));
  if (count && (!grad || !out || (!pre && activation != RST_ACT_NONE)))
    return fail(RST_ERR_INVALID_ARGUMENT, "activation_backward: null operand");
  return launch_act_backward(e->stream, activation, grad, pre, residual, out, count);
}

int rst_linear_act_forward(rst_engine* e, const double* x, const double* weight, const double* bias,
                           const double* residual, double* pre_out, double* out, size_t batch, size_t in_features,
                           size_t out_features, int activation) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_activation("linear_act_forward", activation));
  if (batch == 0 || out_features == 0) return RST_OK;
  if (!out || (in_features && (!x || !weight)))
    return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_forward: null operand");
  RST_TRY(check_dim("linear_act_forward", batch, "batch"));
  RST_TRY(check_dim("linear_act_forward", in_features, "in_features"));
  RST_TRY(check_dim("linear_act_forward", out_features, "out_features"));
  const bool few_rows = linear_rows_supported(batch, out_features, in_features);
  if (!few_rows) RST_TRY(check_contraction(batch, out_features));
  {
    const Range rx{x, batch * in_features}, rw{weight, out_features * in_features}, rb{bias, out_features};
    const Range rr{residual, batch * out_features}, rp{pre_out, batch * out_features}, ro{out, batch * out_features};
    if (overlap_any(ro, {rx, rw, rb, rp}) || overlap_shifted(ro, rr) || overlap_any(rp, {rx, rw, rb, rr}))
      return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_forward: an output over an operand");
  }
  const ActEpilogue act{activation, nullptr, residual, pre_out};
  if (few_rows)
    return launch_linear_rows(e->stream, x, weight, bias, out, act, batch, out_features, in_features);
  GemmDesc d{};
  d.A = x; d.B = weight; d.C = out;
  d.M = (int)batch; d.N = (int)out_features; d.K = (int)in_features;
  d.lda = (long)in_features; d.ldb = (long)in_features; d.ldc = (long)out_features;
  d.a_kc = true; d.b_kc = true;
  d.bias = bias;
  d.epilogue = bias ? EPI_BIAS : EPI_NONE;
  d.workspace = e->d_gemm_ws; d.workspace_count = e->gemm_ws_count;
  if (activation != RST_ACT_NONE || residual || pre_out) d.act = &act;
  return launch_gemm(e->stream, d);
}

int rst_linear_act_backward(rst_engine* e, const double* grad, const double* pre, int activation, double* grad_pre,
                            const double* x, const double* weight, double* grad_weight, double* grad_bias,
                            double* grad_input, const double* input_pre, int input_activation,
                            const double* residual_grad, size_t batch, size_t in_features, size_t out_features) {
  RST_TRY(engine_activate(e));
  RST_TRY(check_activation("linear_act_backward", activation));
  RST_TRY(check_activation("linear_act_backward", input_activation));
  if (batch == 0 || in_features == 0 || out_features == 0)
    return fail(RST_ERR_SHAPE, "linear_act_backward of a batch of %zu through %zu -> %zu features", batch, in_features,
                out_features);
  if (!grad || !x || !weight || !grad_weight)
    return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: null operand");
  if (activation != RST_ACT_NONE && (!pre || !grad_pre))
    return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: an activation needs pre and grad_pre");
  if (grad_input && input_activation != RST_ACT_NONE && !input_pre)
    return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: an input activation needs input_pre");
  RST_TRY(check_dim("linear_act_backward", batch, "batch"));
  RST_TRY(check_dim("linear_act_backward", in_features, "in_features"));
  RST_TRY(check_dim("linear_act_backward", out_features, "out_features"));
  RST_TRY(check_contraction(out_features, in_features));
  if (grad_input) RST_TRY(check_contraction(batch, in_features));
  {
    // what this call reads and writes: grad and pre are read before the products begin, and are free then; the input
    // gradient, while the other gradients are written, reads what both products read, input_pre and residual_grad
    const size_t above = batch * out_features, below = batch * in_features;
    const bool act = activation != RST_ACT_NONE;
    const Range rg{grad, above}, rpre{pre, act ? above : 0}, rdz{act ? grad_pre : grad, above};
    const Range rx{x, below}, rw{weight, grad_input ? in_features * out_features : 0};
    const Range rip{input_pre, grad_input && input_activation != RST_ACT_NONE ? below : 0};
    const Range rres{residual_grad, grad_input ? below : 0};
    const Range ow{grad_weight, in_features * out_features}, ob{grad_bias, out_features}, oi{grad_input, below};
    if (act && (overlap_shifted(rdz, rg) || overlap_shifted(rdz, rpre) || overlap_any(rdz, {rx, rw, rip, rres})))
      return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: grad_pre over what is read after it is written");
    if (overlap_any(ow, {rx, rw, rdz, rip, rres, ob, oi}) || overlap_any(ob, {rx, rw, rdz, rip, rres, oi}))
      return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: a parameter's gradient over another operand");
    if (overlap_any(oi, {rx, rw, rdz}) || overlap_shifted(oi, rip) || overlap_shifted(oi, rres))
      return fail(RST_ERR_INVALID_ARGUMENT, "linear_act_backward: grad_input over x, weight or the products' gradient");
  }
  if (activation != RST_ACT_NONE) {
    RST_TRY(launch_act_backward(e->stream, activation, grad, pre, nullptr, grad_pre, batch * out_features));
    grad = grad_pre;
  }
  const ActEpilogue act{input_activation, input_pre, residual_grad, nullptr};
  return engine_linear_backward(e, grad, x, weight, grad_weight, grad_bias, grad_input, nullptr, &act, batch,
                                in_features, out_features);
}

}  // extern "C"
