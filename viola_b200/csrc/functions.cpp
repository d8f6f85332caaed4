// torch.ops.viola_b200.* with gradients: expert routing (experts.cu) and the RMS norms around a block (block_norm.cu).
//
// Unlike the adapters of bindings.cpp these operators allocate their results and workspaces themselves and are graph
// nodes of their own, written in C++: calls on a few tokens are bound by the host, where a step through Python nodes and
// Python allocations took 115 to 210 us.  A workspace belongs to one call (the caching allocator's, or the capture's
// pool), so neither streams nor captured graphs share one.
// Arguments are checked here too (ValueError, TypeError): in Python the checks of a call took as long as its launch.  The
// same rules for CPU tensors are in viola_b200/nn.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <tuple>
#include <vector>
#include "api.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxExperts = 1024, kMaxTopK = 32, kMaxWidth = 1 << 22;

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int dtype_code(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "expected float32, bfloat16 or float16, got ", t);
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2;
}
void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "viola_b200::", what, " failed: ", cudaGetErrorString((cudaError_t)rc), " (", rc, ")");
}
int narrow(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, name, " out of range: ", v);
  return (int)v;
}
// A tangent would be lost without a word: the plain branches read the values alone, and so do the backward kernels.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... T> void no_tangents(const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), "viola_b200: these operators have no forward-mode derivatives on the GPU");
}
void once_only(const variable_list& grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "viola_b200: the gradients of these operators cannot be differentiated again");
  for (const Tensor& g : grads) no_tangents(g);
}
bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
const Tensor& none() {
  static const Tensor undefined;
  return undefined;
}
const Tensor& value(const OptTensor& t) { return t.has_value() ? *t : none(); }
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
// a CUDA tensor on the device of `like` with unit column stride, as [rows, last dimension]
void on_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device() && t.is_cuda(), name, " is on ", t.device(), ", not on ", like.device());
}
Tensor rows2d(const Tensor& t) {
  Tensor flat = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return flat.stride(1) == 1 ? flat : flat.contiguous();
}
at::DimVector with_last(at::IntArrayRef shape, int64_t last) {
  at::DimVector out(shape.begin(), shape.end());
  out.back() = last;
  return out;
}

// ---- router ----------------------------------------------------------------------------------------------------
struct Routed {
  Tensor flat, weights, indices, counts, balance, z, inverse;
};

Routed route_forward(const Tensor& logits, int64_t top_k, const OptTensor& bias, const OptTensor& mask, bool normalize, bool save) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() >= 1, "logits must be a CUDA tensor with an experts dimension");
  const c10::cuda::CUDAGuard guard(logits.device());
  Routed r;
  const int64_t experts = logits.size(-1);
  const int dtype = dtype_code(logits.scalar_type());
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, "the number of experts must be between 1 and ", kMaxExperts, ", got ", experts);
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= std::min(experts, kMaxTopK), "top_k must be between 1 and min(experts, ", kMaxTopK,
                    "), got ", top_k, " for ", experts, " experts");
  const int tokens = narrow(logits.numel() / experts, "tokens");
  r.flat = tokens > 0 ? rows2d(logits) : logits.reshape({0, experts});
  Tensor offsets, live;
  if (bias.has_value()) {
    on_device(*bias, logits, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == experts, "bias must have shape (", experts, ",), got ", bias->sizes());
    offsets = bias->detach().to(at::kFloat).contiguous();
  }
  if (mask.has_value()) {
    on_device(*mask, logits, "mask");
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->sizes() == logits.sizes().slice(0, logits.dim() - 1),
                      "mask must be bool of the leading shape of logits ", logits.sizes(), ", got ", mask->scalar_type(), " ", mask->sizes());
    live = mask->contiguous();
  }
  const auto f32 = logits.options().dtype(at::kFloat), i32 = logits.options().dtype(at::kInt);
  const at::DimVector shape = with_last(logits.sizes(), top_k);
  r.weights = at::empty(shape, f32);
  r.indices = at::empty(shape, i32);
  r.counts = at::empty({experts}, i32);
  r.balance = at::empty({}, f32);
  r.z = at::empty({}, f32);
  const int64_t need = vb_route_workspace(tokens, experts);
  const Tensor scratch = at::empty({need + (save ? 0 : 2)}, f32);
  if (save) r.inverse = at::empty({2}, f32);
  float* work = scratch.data_ptr<float>();
  check(vb_route_forward(r.flat.data_ptr(), dtype, tokens, (int)experts, r.flat.stride(0), (const float*)ptr(offsets),
                         (const uint8_t*)ptr(live), (int)top_k, normalize, r.weights.data_ptr<float>(),
                         r.indices.data_ptr<int>(), r.counts.data_ptr<int>(), r.balance.data_ptr<float>(),
                         r.z.data_ptr<float>(), save ? r.inverse.data_ptr<float>() : work + need, work, need, stream()),
        "route_forward");
  return r;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t top_k, const OptTensor& bias,
                               const OptTensor& mask, bool normalize) {
    Routed r = route_forward(logits, top_k, bias, mask, normalize, true);
    ctx->save_for_backward({r.flat, r.weights, r.indices, r.counts, r.inverse});
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->mark_non_differentiable({r.indices, r.counts});
    ctx->set_materialize_grads(false);
    return {r.weights, r.indices, r.counts, r.balance, r.z};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only(grads);
    const Tensor &dbalance = grads[3], &dz = grads[4];
    if (!grads[0].defined() && !dbalance.defined() && !dz.defined()) return {none(), none(), none(), none(), none()};
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &flat = saved[0], &indices = saved[2];
    const c10::cuda::CUDAGuard guard(flat.device());
    const Tensor dweights = grads[0].defined() ? grads[0].contiguous() : Tensor();
    Tensor dlogits = at::empty(flat.sizes(), flat.options());
    check(vb_route_backward(flat.data_ptr(), dtype_code(flat.scalar_type()), (int)flat.size(0), (int)flat.size(1), flat.stride(0),
                            (int)ctx->saved_data["top_k"].toInt(), ctx->saved_data["normalize"].toBool(),
                            saved[1].data_ptr<float>(), indices.data_ptr<int>(), saved[3].data_ptr<int>(),
                            saved[4].data_ptr<float>(), (const float*)ptr(dweights), (const float*)ptr(dbalance),
                            (const float*)ptr(dz), dlogits.data_ptr(), stream()),
          "route_backward");
    return {dlogits.view(ctx->saved_data["shape"].toIntVector()), none(), none(), none(), none()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route(const Tensor& logits, int64_t top_k, const OptTensor& bias,
                                                         const OptTensor& mask, bool normalize) {
  no_tangents(logits);         // one of the bias moves nothing
  if (at::GradMode::is_enabled() && wants_grad(logits)) {
    const variable_list out = Route::apply(logits, top_k, bias, mask, normalize);
    return {out[0], out[1], out[2], out[3], out[4]};
  }
  Routed r = route_forward(logits, top_k, bias, mask, normalize, false);
  return {r.weights, r.indices, r.counts, r.balance, r.z};
}

// ---- plan, dispatch, combine -------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> expert_plan(const Tensor& indices, int64_t experts) {
  TORCH_CHECK_TYPE(indices.dim() >= 1 && (indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong),
                   "indices must be int32 or int64 [..., top_k], got ", indices.scalar_type(), " ", indices.sizes());
  TORCH_CHECK_VALUE(indices.is_cuda(), "indices must be a CUDA tensor");
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, "the number of experts must be between 1 and ", kMaxExperts, ", got ", experts);
  TORCH_CHECK_VALUE(indices.size(-1) >= 1 && indices.size(-1) <= kMaxTopK, "indices must hold between 1 and ", kMaxTopK,
                    " choices per token, got ", indices.size(-1));
  const c10::cuda::CUDAGuard guard(indices.device());
  const Tensor flat = indices.contiguous();
  const int n = narrow(flat.numel(), "choices"), e = narrow(experts, "experts");
  const auto i32 = indices.options().dtype(at::kInt);
  Tensor offsets = at::empty({experts + 1}, i32), positions = at::empty({n / indices.size(-1), indices.size(-1)}, i32), workspace;
  const int64_t need = vb_expert_plan_workspace(n, e);
  if (need) workspace = at::empty({need}, i32);
  check(vb_expert_plan(ptr(flat), flat.scalar_type() == at::kLong, n, e, offsets.data_ptr<int>(), positions.data_ptr<int>(),
                       (int*)ptr(workspace), need, stream()),
        "expert_plan");
  return {offsets, positions};
}

struct Plan {
  int tokens, top_k, experts;
  Tensor positions, offsets;
};
Plan check_plan(const Tensor& positions, const Tensor& offsets, const Tensor& like) {
  on_device(positions, like, "positions");
  on_device(offsets, like, "offsets");
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt && positions.dim() == 2 && positions.size(1) >= 1 &&
                    positions.size(1) <= kMaxTopK && offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.numel() >= 2,
                    "plan must hold int32 offsets [experts + 1] and int32 positions [tokens, top_k]");
  narrow(positions.numel(), "choices");
  return {(int)positions.size(0), (int)positions.size(1), narrow(offsets.numel(), "experts") - 1, positions.contiguous(), offsets.contiguous()};
}

Tensor combine_forward(const Tensor& rows, const Tensor& weights, const Tensor& positions, at::IntArrayRef shape) {
  Tensor out = at::empty(shape, rows.options());
  check(vb_expert_combine(ptr(rows), dtype_code(rows.scalar_type()), narrow(rows.size(1), "width"), (int)positions.size(0),
                          (int)positions.size(1), positions.data_ptr<int>(), ptr(weights),
                          weights.defined() ? dtype_code(weights.scalar_type()) : 0, ptr(out), stream()),
        "expert_combine");
  return out;
}

Tensor dispatch_forward(const Tensor& x, const Plan& plan) {
  const Tensor &positions = plan.positions, &offsets = plan.offsets;
  dtype_code(x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxWidth && x.numel() == plan.tokens * x.size(-1),
                    "x of shape ", x.sizes(), " does not hold the plan's ", plan.tokens, " tokens");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t width = x.size(-1);
  const Tensor flat = plan.tokens ? rows2d(x) : x.reshape({0, width});
  Tensor rows = at::empty({positions.numel(), width}, x.options());
  check(vb_expert_dispatch(ptr(flat), flat.stride(0) * flat.element_size(), width * flat.element_size(), plan.tokens, plan.top_k,
                           positions.data_ptr<int>(), offsets.data_ptr<int>(), plan.experts, ptr(rows), stream()),
        "expert_dispatch");
  return rows;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& offsets) {
    const Plan plan = check_plan(positions, offsets, x);
    ctx->save_for_backward({plan.positions});
    ctx->saved_data["shape"] = x.sizes().vec();
    return dispatch_forward(x, plan);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only(grads);
    const variable_list saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    return {combine_forward(grads[0].contiguous(), none(), saved[0], ctx->saved_data["shape"].toIntVector()), none(), none()};
  }
};

Tensor expert_dispatch(const Tensor& x, const Tensor& positions, const Tensor& offsets) {
  no_tangents(x);
  if (at::GradMode::is_enabled() && wants_grad(x)) return Dispatch::apply(x, positions, offsets);
  return dispatch_forward(x, check_plan(positions, offsets, x));
}

Plan check_combine(const Tensor& rows, const Tensor& weights, const Tensor& positions, const Tensor& offsets) {
  const Plan plan = check_plan(positions, offsets, rows);
  on_device(weights, rows, "weights");
  dtype_code(rows.scalar_type());
  dtype_code(weights.scalar_type());
  TORCH_CHECK_VALUE(rows.dim() == 2 && rows.size(0) == positions.numel() && rows.size(1) >= 1 && rows.size(1) <= kMaxWidth,
                    "rows must be [", positions.numel(), ", width], got ", rows.sizes());
  TORCH_CHECK_VALUE(weights.dim() >= 1 && weights.size(-1) == plan.top_k && weights.numel() == positions.numel(),
                    "weights of shape ", weights.sizes(), " do not match the plan's ", plan.tokens, " tokens x ", plan.top_k, " choices");
  return plan;
}

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& positions, const Tensor& offsets) {
    const c10::cuda::CUDAGuard guard(rows.device());
    const Tensor r = rows.contiguous(), w = weights.contiguous();
    ctx->save_for_backward({r, w, positions, offsets});
    return combine_forward(r, w, positions, with_last(weights.sizes(), rows.size(1)));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only(grads);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &weights = saved[1], &positions = saved[2], &offsets = saved[3];
    const c10::cuda::CUDAGuard guard(rows.device());
    const Tensor dout = grads[0].contiguous();
    Tensor drows, dweights;
    if (ctx->needs_input_grad(0)) drows = at::empty(rows.sizes(), rows.options());
    if (ctx->needs_input_grad(1)) dweights = at::empty(weights.sizes(), weights.options());
    check(vb_expert_combine_backward(ptr(dout), ptr(rows), dtype_code(rows.scalar_type()), (int)rows.size(1),
                                     (int)positions.size(0), (int)positions.size(1), positions.data_ptr<int>(),
                                     offsets.data_ptr<int>(), (int)offsets.numel() - 1, ptr(weights),
                                     dtype_code(weights.scalar_type()), ptr(drows), ptr(dweights), stream()),
          "expert_combine_backward");
    return {drows, dweights, none(), none()};
  }
};

Tensor expert_combine(const Tensor& rows, const Tensor& weights, const Tensor& positions, const Tensor& offsets) {
  no_tangents(rows, weights);
  const Plan plan = check_combine(rows, weights, positions, offsets);
  if (at::GradMode::is_enabled() && (wants_grad(rows) || wants_grad(weights)))
    return Combine::apply(rows, weights, plan.positions, plan.offsets);
  const c10::cuda::CUDAGuard guard(rows.device());
  return combine_forward(rows.contiguous(), weights.contiguous(), plan.positions, with_last(weights.sizes(), rows.size(1)));
}

// ---- RMS norms around a block --------------------------------------------------------------------------------------
// [cols]: shared by all rows; [batch, cols] where `samples`: one row per sample; what the kernels cannot read in place is copied
Tensor vector_in_place(const OptTensor& t, const Tensor& x, bool samples, const char* name) {
  if (!t.has_value()) return Tensor();
  on_device(*t, x, name);
  dtype_code(t->scalar_type());
  const int64_t cols = x.size(-1);
  const bool per_sample = samples && x.dim() >= 2 && t->dim() == 2 && t->size(0) == x.size(0) && t->size(1) == cols;
  TORCH_CHECK_VALUE(per_sample || (t->dim() == 1 && t->size(0) == cols), name, " must have shape (", cols, ",)",
                    samples ? " or (batch, width)" : "", " for x of shape ", x.sizes(), ", got ", t->sizes());
  const bool rows_apart = t->dim() == 1 || t->size(0) == 1 || t->stride(0) >= cols;
  return (t->stride(-1) == 1 || cols == 1) && rows_apart ? *t : t->contiguous();
}
VbNormVector norm_vector(const Tensor& t) {
  if (!t.defined()) return VbNormVector{nullptr, 0, 0};
  const int64_t pitch = t.dim() == 1 ? 0 : t.size(0) == 1 ? t.size(1) : t.stride(0);
  return VbNormVector{t.data_ptr(), dtype_code(t.scalar_type()), pitch};
}

struct Normed {
  Tensor x, y, weight, gate, next_weight, next_scale, out, h, ry, ru;
  int64_t tokens = 0;
  VbBlockNorm args{};
};

VbBlockNorm norm_args(const Normed& n, int64_t rows, int64_t cols, int64_t tokens, double residual_scale, double eps, int y_dtype) {
  VbBlockNorm a{};
  a.rows = narrow(rows, "rows");
  a.cols = narrow(cols, "cols");
  a.tokens = narrow(tokens, "tokens");
  a.x_dtype = dtype_code(n.x.scalar_type());
  a.y_dtype = y_dtype;
  a.residual_scale = (float)residual_scale;
  a.eps = (float)eps;
  a.x = ptr(n.x);
  a.y = ptr(n.y);
  a.weight = norm_vector(n.weight);
  a.gate = norm_vector(n.gate);
  a.next_weight = norm_vector(n.next_weight);
  a.next_scale = norm_vector(n.next_scale);
  a.ry = (float*)ptr(n.ry);
  a.ru = (float*)ptr(n.ru);
  return a;
}

// h_dtype: -1 for no h, else a dtype code
Normed norm_forward(const Tensor& x, const OptTensor& y, const OptTensor& weight, const OptTensor& gate, const OptTensor& next_weight,
                    const OptTensor& next_scale, double residual_scale, double eps, int64_t h_dtype, bool save) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && x.numel() > 0 && x.size(-1) <= VB_NORM_MAX_COLS,
                    "the width must be between 1 and ", VB_NORM_MAX_COLS, ", got x of shape ", x.sizes());
  dtype_code(x.scalar_type());
  constexpr double most = std::numeric_limits<float>::max(), least = std::numeric_limits<float>::min();
  TORCH_CHECK_VALUE(eps >= least && eps <= most, "eps must be a positive fp32 number, got ", eps);
  TORCH_CHECK_VALUE(std::abs(residual_scale) <= most, "residual_scale must be a finite fp32 number, got ", residual_scale);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  Normed n;
  n.x = x.contiguous();
  if (y.has_value()) {
    on_device(*y, x, "y");
    TORCH_CHECK_VALUE(y->sizes() == x.sizes(), "y must have the shape of x, got ", y->sizes(), " and ", x.sizes());
    dtype_code(y->scalar_type());
    TORCH_CHECK_TYPE(x.scalar_type() == at::kFloat || x.scalar_type() == y->scalar_type(),
                     "x must be float32 or have the dtype of y, got ", x.scalar_type(), " and ", y->scalar_type());
    n.y = y->contiguous();
    n.out = at::empty(x.sizes(), x.options());
  }
  n.weight = vector_in_place(weight, x, false, "weight");
  n.gate = vector_in_place(gate, x, true, "gate");
  n.next_weight = vector_in_place(next_weight, x, false, y.has_value() ? "next_weight" : "weight");
  n.next_scale = vector_in_place(next_scale, x, true, y.has_value() ? "next_scale" : "scale");
  // rows of a sample (all rows where no vector is per sample)
  const bool per_sample = (n.gate.defined() && n.gate.dim() == 2) || (n.next_scale.defined() && n.next_scale.dim() == 2);
  n.tokens = per_sample ? rows / x.size(0) : rows;
  const auto f32 = x.options().dtype(at::kFloat);
  if (h_dtype >= 0) n.h = at::empty(x.sizes(), x.options().dtype(h_dtype == 0 ? at::kFloat : h_dtype == 1 ? at::kBFloat16 : at::kHalf));
  if (save && n.y.defined()) n.ry = at::empty({rows}, f32);
  if (save && n.h.defined()) n.ru = at::empty({rows}, f32);
  const int y_dtype = n.y.defined() ? dtype_code(n.y.scalar_type()) : (int)h_dtype;
  TORCH_CHECK_TYPE(h_dtype < 0 || h_dtype == y_dtype, "viola_b200: h has the dtype of y");
  n.args = norm_args(n, rows, cols, n.tokens, residual_scale, eps, y_dtype);
  n.args.out = ptr(n.out);
  n.args.h = ptr(n.h);
  check(vb_block_norm(&n.args, stream()), "block_norm");
  return n;
}

variable_list norm_results(const Normed& n) {
  if (!n.out.defined()) return {n.h};
  if (!n.h.defined()) return {n.out};
  return {n.out, n.h};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& y, const OptTensor& weight,
                               const OptTensor& gate, const OptTensor& next_weight, const OptTensor& next_scale,
                               double residual_scale, double eps, int64_t h_dtype) {
    const Normed n = norm_forward(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, h_dtype, true);
    ctx->save_for_backward({n.x, n.y, n.weight, n.gate, n.next_weight, n.next_scale, n.ry, n.ru});
    ctx->saved_data["tokens"] = n.tokens;
    ctx->saved_data["residual_scale"] = residual_scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["y_dtype"] = (int64_t)n.args.y_dtype;
    ctx->set_materialize_grads(false);
    return norm_results(n);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only(grads);
    variable_list result(9);
    const variable_list saved = ctx->get_saved_variables();
    Normed n;
    n.x = saved[0]; n.y = saved[1]; n.weight = saved[2]; n.gate = saved[3];
    n.next_weight = saved[4]; n.next_scale = saved[5]; n.ry = saved[6]; n.ru = saved[7];
    const bool post = n.y.defined(), pre = n.ru.defined();
    Tensor dout, dh;
    if (post && grads[0].defined()) dout = grads[0].contiguous();
    if (pre && grads[post ? 1 : 0].defined()) dh = grads[post ? 1 : 0].contiguous();
    if (!dout.defined() && !dh.defined()) return result;
    const c10::cuda::CUDAGuard guard(n.x.device());
    const int64_t cols = n.x.size(-1), rows = n.x.numel() / cols, tokens = ctx->saved_data["tokens"].toInt();
    VbBlockNorm a = norm_args(n, rows, cols, tokens, ctx->saved_data["residual_scale"].toDouble(), ctx->saved_data["eps"].toDouble(),
                              (int)ctx->saved_data["y_dtype"].toInt());
    const Tensor* sources[6] = {&n.x, &n.y, &n.weight, &n.gate, &n.next_weight, &n.next_scale};
    const bool reached[6] = {true, post, post, post, dh.defined(), dh.defined()};
    bool sums = false;
    size_t at_input = 0;       // needs_input_grad counts the tensor inputs that are there
    for (int i = 0; i < 6; ++i) {
      if (!sources[i]->defined()) continue;
      if (ctx->needs_input_grad(at_input++) && reached[i]) {
        result[i] = at::empty(sources[i]->sizes(), sources[i]->options());
        sums = sums || i >= 2;
      }
    }
    VbBlockNormGrads g{};
    g.dout = ptr(dout); g.dh = ptr(dh);
    g.dx = ptr(result[0]); g.dy = ptr(result[1]);
    g.dweight = ptr(result[2]); g.dgate = ptr(result[3]);
    g.dnext_weight = ptr(result[4]); g.dnext_scale = ptr(result[5]);
    Tensor workspace;
    if (sums) {
      g.workspace_floats = vb_block_norm_workspace((int)rows, (int)cols, (int)tokens);
      workspace = at::empty({(int64_t)g.workspace_floats}, n.x.options().dtype(at::kFloat));
      g.workspace = workspace.data_ptr<float>();
    }
    check(vb_block_norm_backward(&a, &g, stream()), "block_norm_backward");
    return result;
  }
};

std::vector<Tensor> block_norm(const Tensor& x, const OptTensor& y, const OptTensor& weight, const OptTensor& gate,
                               const OptTensor& next_weight, const OptTensor& next_scale, double residual_scale, double eps,
                               int64_t h_dtype) {
  no_tangents(x, y, weight, gate, next_weight, next_scale);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(y) || wants_grad(weight) || wants_grad(gate) ||
                                     wants_grad(next_weight) || wants_grad(next_scale)))
    return BlockNorm::apply(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, h_dtype);
  return norm_results(norm_forward(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, h_dtype, false));
}

int64_t block_launches() { return vb_block_launches(); }

}  // namespace

TORCH_LIBRARY_FRAGMENT(viola_b200, m) {
  m.def("route", &route);
  m.def("expert_plan", &expert_plan);
  m.def("expert_dispatch", &expert_dispatch);
  m.def("expert_combine", &expert_combine);
  m.def("block_norm", &block_norm);
  m.def("block_launches", &block_launches);
}
