// The feed-forward operators (layer norm, dense layers, plans of groups) as operators of libtorch's dispatcher,
// with their autograd nodes, over the C ABI (host code); as attention_ops.cpp, whose header they share.
#define XNN_ENTRIES(X)                                                                           \
  X(xnn_last_error) X(xnn_layer_norm) X(xnn_layer_norm_backward_work_size)                       \
  X(xnn_layer_norm_backward) X(xnn_group_plan_size) X(xnn_group_plan) X(xnn_linear)              \
  X(xnn_linear_work_size) X(xnn_linear_backward_work_size) X(xnn_linear_backward)
#define XNN_FAMILY "feed-forward"

#include "native_ops.h"

namespace {

typedef std::tuple<Tensor, Tensor> Two;
typedef std::tuple<Tensor, Tensor, Tensor> Three;

// ---------------------------------------------------------------- rows
// x as rows of its last dimension, with unit stride and no overlap; a view where its layout allows
Tensor as_rows(const Tensor& x) {
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1))) r = r.contiguous();
  return r;
}
int64_t row_stride(const Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

void check_rows(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be (..., width) with width at least 1, got ",
                    x.sizes());
}

// an optional operand of x's type and of these sizes
void check_like(const Tensor& t, const Tensor& x, at::IntArrayRef sizes, const char* name) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " is ", t.scalar_type(), ", x is ",
                   x.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must be ", sizes, ", got ", t.sizes());
}

Tensor contiguous(const MaybeTensor& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }

Tensor empty_if(bool wanted, at::IntArrayRef sizes, const Tensor& like) {
  return wanted ? at::empty(sizes, like.options()) : at::empty({0}, like.options());
}
Tensor empty_shape(bool wanted, const Tensor& like) {
  return wanted ? at::empty_symint(like.sym_sizes(), like.options()) : at::empty({0}, like.options());
}
void* data_if(bool wanted, const Tensor& t) { return wanted ? t.data_ptr() : nullptr; }

// ---------------------------------------------------------------- layer norm
#define XNN_NORM_ARGUMENTS const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps
#define XNN_NORM_TYPES const Tensor&, const MaybeTensor&, const MaybeTensor&, double

Tensor layer_norm(XNN_NORM_ARGUMENTS) {
  XNN_OPERATOR("layer_norm", Tensor(XNN_NORM_TYPES));
  return op.call(x, weight, bias, eps);
}

// with the rows' means and reciprocal deviations
Two layer_norm_stats(XNN_NORM_ARGUMENTS) {
  XNN_OPERATOR("layer_norm_stats", Two(XNN_NORM_TYPES));
  return op.call(x, weight, bias, eps);
}

// the gradients of x, weight and bias; those that are not wanted are empty
Three layer_norm_backward(const Tensor& grad, const Tensor& x, const MaybeTensor& weight, const Tensor& stats,
                          bool input, bool weights, bool biases) {
  XNN_OPERATOR("layer_norm_backward",
               Three(const Tensor&, const Tensor&, const MaybeTensor&, const Tensor&, bool, bool, bool));
  return op.call(grad, x, weight, stats, input, weights, biases);
}

Two layer_norm_forward(XNN_NORM_ARGUMENTS, bool keep) {
  const Tensor w = contiguous(weight), b = contiguous(bias);
  check_tensors({&x, &w, &b});
  check_rows(x);
  const int code = storage_code(x);
  check_like(w, x, {x.size(-1)}, "weight");
  check_like(b, x, {x.size(-1)}, "bias");
  TORCH_CHECK_VALUE(eps >= 0.0 && eps < std::numeric_limits<double>::infinity(),
                    "eps must be finite and not negative, got ", eps);
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x);
  Tensor out = at::empty(x.sizes(), x.options()), stats;
  if (keep) stats = at::empty({rows.size(0), 2}, x.options().dtype(at::kFloat));
  XNN_CALL(xnn_layer_norm, code, data(rows), row_stride(rows), rows.size(0), (int32_t)rows.size(1), data(w),
           data(b), (float)eps, data(out), (float*)data(stats), stream_of(x));
  return {out, stats};
}

Tensor layer_norm_kernel(XNN_NORM_ARGUMENTS) { return std::get<0>(layer_norm_forward(x, weight, bias, eps, false)); }
Two layer_norm_stats_kernel(XNN_NORM_ARGUMENTS) { return layer_norm_forward(x, weight, bias, eps, true); }

c10::SymInt rows_of(const Tensor& x) {
  c10::SymInt n = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) n = n * x.sym_size(d);
  return n;
}

Tensor layer_norm_shape(const Tensor& x, const MaybeTensor&, const MaybeTensor&, double) {
  return at::empty_symint(x.sym_sizes(), x.options());
}
Two layer_norm_stats_shape(const Tensor& x, const MaybeTensor&, const MaybeTensor&, double) {
  return {at::empty_symint(x.sym_sizes(), x.options()),
          at::empty_symint({rows_of(x), 2}, x.options().dtype(at::kFloat))};
}

Three layer_norm_backward_kernel(const Tensor& grad_, const Tensor& x, const MaybeTensor& weight,
                                 const Tensor& stats_, bool input, bool weights, bool biases) {
  const Tensor w = contiguous(weight);
  check_tensors({&x, &grad_, &w, &stats_});
  check_rows(x);
  const int code = storage_code(x);
  check_like(w, x, {x.size(-1)}, "weight");
  check_like(grad_, x, x.sizes(), "the cotangent");
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), grad = grad_.contiguous(), stats = stats_.contiguous();
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == rows.size(0) &&
                        stats.size(1) == 2,
                    "statistics ", stats.sizes(), " ", stats.scalar_type(), " of ", rows.size(0), " rows");
  const Tensor dx = empty_if(input, x.sizes(), x), dw = empty_if(weights, {x.size(-1)}, x),
               db = empty_if(biases, {x.size(-1)}, x);
  Tensor work;
  size_t need = 0;
  if (weights || biases) {
    check("xnn_layer_norm_backward_work_size",
          api.xnn_layer_norm_backward_work_size((int32_t)rows.size(1), &need));
    work = bytes(x, need);
  }
  XNN_CALL(xnn_layer_norm_backward, code, data(grad), data(rows), row_stride(rows), rows.size(0),
           (int32_t)rows.size(1), data(w), (const float*)data(stats), data_if(input, dx), data_if(weights, dw),
           data_if(biases, db), data(work), need, stream_of(x));
  return {dx, dw, db};
}

Three layer_norm_backward_shape(const Tensor&, const Tensor& x, const MaybeTensor&, const Tensor&, bool input,
                                bool weights, bool biases) {
  const auto row = [&](bool wanted) {
    return wanted ? at::empty_symint({x.sym_size(-1)}, x.options()) : at::empty({0}, x.options());
  };
  return {empty_shape(input, x), row(weights), row(biases)};
}

struct LayerNormBackward : Node {
  SavedVariable x, weight, stats;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable();
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const bool wanted[] = {task_should_compute_output(0), task_should_compute_output(1),
                           task_should_compute_output(2)};
    // unpacked first: a checkpoint computes the forward pass again then, with its derivatives
    const Tensor x_ = x.unpack(), weight_ = wanted[0] ? weight.unpack() : Tensor(), stats_ = stats.unpack();
    at::AutoDispatchBelowADInplaceOrView below;            // no derivative of its own
    const Three all = layer_norm_backward(grads[0], x_, maybe(weight_), stats_, wanted[0], wanted[1], wanted[2]);
    if (wanted[0]) out[0] = std::get<0>(all);
    if (wanted[1]) out[1] = std::get<1>(all);
    if (wanted[2]) out[2] = std::get<2>(all);
    return out;
  }
  void release_variables() override {
    for (SavedVariable* v : {&x, &weight, &stats}) v->reset_data();
  }
  std::string name() const override { return "XnnLayerNormBackward"; }
};

Tensor layer_norm_autograd(XNN_NORM_ARGUMENTS) {
  const Tensor w = or_none(weight), b = or_none(bias);
  refuse_tangents({&x, &w, &b});
  if (!wanted({&x, &w, &b})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm(x, weight, bias, eps);
  }
  Tensor out, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(out, stats) = layer_norm_stats(x, weight, bias, eps);
  }
  auto node = node_of<LayerNormBackward>(x, w, b);
  node->x = SavedVariable(x, false);
  if (x.requires_grad()) node->weight = SavedVariable(w, false);   // of dx alone
  node->stats = SavedVariable(stats, false);
  set_history(out, node);
  return out;
}

// ---------------------------------------------------------------- groups
Tensor group_plan(const Tensor& ids, int64_t n_groups) {
  XNN_OPERATOR("group_plan", Tensor(const Tensor&, int64_t));
  return op.call(ids, n_groups);
}

Tensor group_plan_kernel(const Tensor& ids_, int64_t n_groups) {
  check_tensors({&ids_});
  check_integers(ids_, "ids");
  TORCH_CHECK_VALUE(ids_.dim() == 1, "ids must be (rows,), got ", ids_.sizes());
  TORCH_CHECK_VALUE(n_groups >= 1 && n_groups <= std::numeric_limits<int32_t>::max(),
                    "n_groups must be positive, got ", n_groups);
  const c10::DeviceGuard guard(ids_.device());
  const Tensor ids = as_int64(ids_);
  size_t plan_bytes = 0, need = 0;
  check("xnn_group_plan_size", api.xnn_group_plan_size(ids.numel(), (int32_t)n_groups, &plan_bytes, &need));
  Tensor plan = at::empty({(int64_t)(plan_bytes / sizeof(int32_t))}, ids.options().dtype(at::kInt));
  const Tensor work = bytes(ids, need);
  XNN_CALL(xnn_group_plan, ids.const_data_ptr<int64_t>(), ids.numel(), (int32_t)n_groups,
           plan.data_ptr<int32_t>(), data(work), need, stream_of(ids));
  return plan;
}

// as xnn_group_plan_size: the rows, where the groups begin, and fifty-two lists of their tiles
constexpr int kPlanLists = 53;
Tensor group_plan_shape(const Tensor& ids, int64_t n_groups) {
  return at::empty_symint({ids.sym_numel() + kPlanLists * (n_groups + 2)}, ids.options().dtype(at::kInt));
}
template <typename N>
N groups_of(const N& plan, const N& rows) {
  return (plan - rows) / kPlanLists - 2;
}

// ---------------------------------------------------------------- dense layers
#define XNN_DENSE_ARGUMENTS                                                                     \
  const Tensor &x, const Tensor &weight, const MaybeTensor &bias, int64_t activation,           \
      const MaybeTensor &residual, const MaybeTensor &plan
#define XNN_DENSE_TYPES \
  const Tensor&, const Tensor&, const MaybeTensor&, int64_t, const MaybeTensor&, const MaybeTensor&

Tensor dense(XNN_DENSE_ARGUMENTS) {
  XNN_OPERATOR("dense", Tensor(XNN_DENSE_TYPES));
  return op.call(x, weight, bias, activation, residual, plan);
}

// with the activation's derivative
Two dense_slope(XNN_DENSE_ARGUMENTS) {
  XNN_OPERATOR("dense_slope", Two(XNN_DENSE_TYPES));
  return op.call(x, weight, bias, activation, residual, plan);
}

// the gradients of x, weight and bias; those that are not wanted are empty
// (x is needed for the last two alone, weight for the first)
Three dense_backward(const Tensor& grad, const MaybeTensor& slope, const MaybeTensor& x, const MaybeTensor& weight,
                     const MaybeTensor& plan, bool input, bool weights, bool biases) {
  XNN_OPERATOR("dense_backward", Three(const Tensor&, const MaybeTensor&, const MaybeTensor&, const MaybeTensor&,
                                       const MaybeTensor&, bool, bool, bool));
  return op.call(grad, slope, x, weight, plan, input, weights, biases);
}

// the slope's own form: float32, float16 beside bfloat16, 16 bits of its own beside float16
at::ScalarType slope_type(const Tensor& x) {
  return x.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type() == at::kBFloat16 ? at::kHalf : at::kShort;
}

// the sizes of an operation's operands
struct Dense {
  int64_t rows, n_in, n_out, groups;
  std::vector<int64_t> out, bias;
};

void check_sizes(const Dense& d, const Tensor& plan) {
  if (plan.defined()) {
    TORCH_CHECK_VALUE(d.groups >= 1, "no groups");
    size_t plan_bytes = 0, need = 0;
    check("xnn_group_plan_size",
          api.xnn_group_plan_size(d.rows, (int32_t)std::min<int64_t>(d.groups, 1 << 30), &plan_bytes, &need));
    TORCH_CHECK_VALUE(plan.scalar_type() == at::kInt && plan.dim() == 1 && plan.is_contiguous() &&
                          plan.size(0) == (int64_t)(plan_bytes / sizeof(int32_t)),
                      "the plan is not of ", d.rows, " rows and ", d.groups, " groups");
  }
  TORCH_CHECK_VALUE(d.n_in < (1 << 20) && d.n_out < (1 << 20), "widths must be below 2^20, got ", d.n_in, " and ",
                    d.n_out);
}

Dense check_dense(const Tensor& x, const Tensor& weight, const Tensor& plan) {
  check_rows(x);
  storage_code(x);
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "weight is ", weight.scalar_type(), ", x is ",
                   x.scalar_type());
  const int64_t lead = plan.defined() ? 1 : 0;
  TORCH_CHECK_VALUE(weight.dim() == 2 + lead && weight.size(lead) == x.size(-1) && weight.size(-1) >= 1,
                    "weight must be (", lead ? "groups, " : "", x.size(-1), ", outputs) for x ", x.sizes(), ", got ",
                    weight.sizes());
  Dense d;
  d.n_in = x.size(-1);
  d.n_out = weight.size(-1);
  d.rows = x.numel() / d.n_in;
  d.groups = lead ? weight.size(0) : 1;
  d.out = x.sizes().vec();
  d.out.back() = d.n_out;
  if (lead) d.bias.push_back(d.groups);
  d.bias.push_back(d.n_out);
  check_sizes(d, plan);
  return d;
}

Two dense_forward(XNN_DENSE_ARGUMENTS, bool keep) {
  const Tensor b = contiguous(bias), r = contiguous(residual), p = or_none(plan);
  check_tensors({&x, &weight, &b, &r, &p});
  const Dense d = check_dense(x, weight, p);
  check_like(b, x, d.bias, "bias");
  check_like(r, x, d.out, "residual");
  TORCH_CHECK_VALUE(activation >= XNN_NO_ACTIVATION && activation <= XNN_TANH, "unknown activation ", activation);
  const c10::DeviceGuard guard(x.device());
  const Tensor rows = as_rows(x), w = weight.contiguous();
  Tensor out = at::empty(d.out, x.options()), slope;
  if (keep)
    slope = at::empty(activation != XNN_NO_ACTIVATION ? at::IntArrayRef(d.out) : at::IntArrayRef({0}),
                      x.options().dtype(slope_type(x)));
  Tensor work;
  size_t need = 0;
  check("xnn_linear_work_size", api.xnn_linear_work_size(storage_code(x), d.rows, (int32_t)d.n_in, (int32_t)d.n_out,
                                                         (int32_t)d.groups, p.defined(), &need));
  if (need > 0) work = bytes(x, need);
  XNN_CALL(xnn_linear, storage_code(x), data(rows), row_stride(rows), d.rows, (int32_t)d.n_in, (int32_t)d.n_out,
           data(w), data(b), (int32_t)activation, data(r), (const int32_t*)data(p), (int32_t)d.groups, data(out),
           data_if(keep && activation != XNN_NO_ACTIVATION, slope), data(work), need, stream_of(x));
  return {out, slope};
}

Tensor dense_kernel(XNN_DENSE_ARGUMENTS) {
  return std::get<0>(dense_forward(x, weight, bias, activation, residual, plan, false));
}
Two dense_slope_kernel(XNN_DENSE_ARGUMENTS) {
  return dense_forward(x, weight, bias, activation, residual, plan, true);
}

Tensor dense_shape(XNN_DENSE_ARGUMENTS) {
  auto sizes = x.sym_sizes().vec();
  sizes.back() = weight.sym_size(-1);
  return at::empty_symint(sizes, x.options());
}
Two dense_slope_shape(XNN_DENSE_ARGUMENTS) {
  const Tensor out = dense_shape(x, weight, bias, activation, residual, plan);
  const auto options = x.options().dtype(slope_type(x));
  return {out, activation != XNN_NO_ACTIVATION ? at::empty_symint(out.sym_sizes(), options) : at::empty({0}, options)};
}

// the operation's sizes from the cotangent and one of x and the weight
Dense check_one(const Tensor& grad, const Tensor& x, const Tensor& weight, const Tensor& plan) {
  Dense d;
  check_rows(grad);
  if (x.defined()) check_rows(x);
  TORCH_CHECK_VALUE(!weight.defined() || weight.dim() == (plan.defined() ? 3 : 2), "weight must be (",
                    plan.defined() ? "groups, " : "", "inputs, outputs), got ", weight.sizes());
  d.n_in = x.defined() ? x.size(-1) : weight.size(-2);
  d.n_out = grad.size(-1);
  d.rows = grad.numel() / d.n_out;
  d.groups = !plan.defined() ? 1 : weight.defined() ? weight.size(0) : groups_of(plan.numel(), d.rows);
  d.out = grad.sizes().vec();
  if (plan.defined()) d.bias.push_back(d.groups);
  d.bias.push_back(d.n_out);
  check_sizes(d, plan);
  return d;
}

Three dense_backward_kernel(const Tensor& grad_, const MaybeTensor& slope_, const MaybeTensor& x_,
                            const MaybeTensor& weight_, const MaybeTensor& plan, bool input, bool weights,
                            bool biases) {
  const Tensor slope = contiguous(slope_), p = or_none(plan), x = or_none(x_), weight = or_none(weight_);
  check_tensors({&grad_, &x, &slope, &weight, &p});
  weights = weights || biases;                             // the weight's product has the bias's sums
  TORCH_CHECK_VALUE(x.defined() || !weights, "the weight's and the bias's gradients need x");
  TORCH_CHECK_VALUE(weight.defined() || !input, "x's gradient needs the weight");
  const int code = storage_code(grad_);
  if (!input && !weights) return {empty_if(false, {}, grad_), empty_if(false, {}, grad_), empty_if(false, {}, grad_)};
  const Dense d = x.defined() && weight.defined() ? check_dense(x, weight, p) : check_one(grad_, x, weight, p);
  std::vector<int64_t> in = d.out, shape = d.bias;
  in.back() = d.n_in;
  shape.insert(shape.end() - 1, d.n_in);
  check_like(grad_, x.defined() ? x : weight, d.out, "the cotangent");
  TORCH_CHECK_VALUE(!x.defined() || x.sizes() == in, "x must be ", in, ", got ", x.sizes());
  TORCH_CHECK_VALUE(!weight.defined() || weight.sizes() == shape, "weight must be ", shape, ", got ", weight.sizes());
  TORCH_CHECK_VALUE(!slope.defined() || (slope.sizes() == d.out && slope.scalar_type() == slope_type(grad_)),
                    "the slope is not that of the forward pass");
  const c10::DeviceGuard guard(grad_.device());
  const Tensor rows = x.defined() ? as_rows(x) : Tensor(), w = contiguous(weight_), grad = grad_.contiguous();
  const Tensor dx = empty_if(input, in, grad), dw = empty_if(weights, shape, grad), db = empty_if(biases, d.bias, grad);
  Tensor work;
  size_t need = 0;
  check("xnn_linear_backward_work_size",
        api.xnn_linear_backward_work_size(code, d.rows, (int32_t)d.n_in, (int32_t)d.n_out, (int32_t)d.groups,
                                          p.defined(), slope.defined(), input, weights, biases, &need));
  if (need > 0) work = bytes(grad, need);
  XNN_CALL(xnn_linear_backward, code, data(grad), data(slope), data(rows), x.defined() ? row_stride(rows) : d.n_in,
           d.rows, (int32_t)d.n_in, (int32_t)d.n_out, data(w), (const int32_t*)data(p), (int32_t)d.groups,
           data_if(input, dx), data_if(weights, dw), data_if(biases, db), data(work), need, stream_of(grad));
  return {dx, dw, db};
}

Three dense_backward_shape(const Tensor& grad, const MaybeTensor&, const MaybeTensor& x_, const MaybeTensor& weight_,
                           const MaybeTensor& plan_, bool input, bool weights, bool biases) {
  const Tensor x = or_none(x_), weight = or_none(weight_), plan = or_none(plan_);
  const auto none = [&] { return at::empty({0}, grad.options()); };
  if (!x.defined() && !weight.defined()) return {none(), none(), none()};
  const c10::SymInt n_in = x.defined() ? x.sym_size(-1) : weight.sym_size(-2);
  std::vector<c10::SymInt> bias, in = grad.sym_sizes().vec();
  if (plan.defined())
    bias.push_back(weight.defined() ? weight.sym_size(0) : groups_of(plan.sym_numel(), rows_of(grad)));
  bias.push_back(grad.sym_size(-1));
  std::vector<c10::SymInt> shape = bias;
  shape.insert(shape.end() - 1, n_in);
  in.back() = n_in;
  return {input ? at::empty_symint(in, grad.options()) : none(),
          weights || biases ? at::empty_symint(shape, grad.options()) : none(),
          biases ? at::empty_symint(bias, grad.options()) : none()};
}

struct DenseBackward : Node {
  SavedVariable x, weight, slope, plan;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const bool wanted[] = {task_should_compute_output(0), task_should_compute_output(1),
                           task_should_compute_output(2)};
    if (task_should_compute_output(3)) out[3] = grads[0];
    if (!wanted[0] && !wanted[1] && !wanted[2]) return out;
    once_differentiable();
    // Unpacked first: a checkpoint computes the forward pass again then, with its derivatives. (Unpacking asks whether a
    // tensor was written to: only of those that these gradients need.)
    const Tensor slope_ = slope.unpack(), plan_ = plan.unpack();
    const Tensor x_ = wanted[1] || wanted[2] ? x.unpack() : Tensor(), weight_ = wanted[0] ? weight.unpack() : Tensor();
    at::AutoDispatchBelowADInplaceOrView below;            // no derivative of its own
    const Three all = dense_backward(grads[0], maybe(slope_), maybe(x_), maybe(weight_), maybe(plan_), wanted[0],
                                     wanted[1], wanted[2]);
    if (wanted[0]) out[0] = std::get<0>(all);
    if (wanted[1]) out[1] = std::get<1>(all);
    if (wanted[2]) out[2] = std::get<2>(all);
    return out;
  }
  void release_variables() override {
    for (SavedVariable* v : {&x, &weight, &slope, &plan}) v->reset_data();
  }
  std::string name() const override { return "XnnDenseBackward"; }
};

Tensor dense_autograd(XNN_DENSE_ARGUMENTS) {
  const Tensor b = or_none(bias), r = or_none(residual), p = or_none(plan);
  refuse_tangents({&x, &weight, &b, &r});
  const bool product = wanted({&x, &weight, &b}) && activation != XNN_NO_ACTIVATION;
  Tensor out, slope;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (product)
      std::tie(out, slope) = dense_slope(x, weight, bias, activation, residual, plan);
    else
      out = dense(x, weight, bias, activation, residual, plan);
  }
  if (!wanted({&x, &weight, &b, &r})) return out;
  auto node = node_of<DenseBackward>(x, weight, b, r);
  if (wanted({&weight, &b})) node->x = SavedVariable(x, false);
  if (x.requires_grad()) node->weight = SavedVariable(weight, false);
  node->slope = SavedVariable(slope, false);
  node->plan = SavedVariable(p, false);
  set_history(out, node);
  return out;
}

#define XNN_NORM_SCHEMA "Tensor x, Tensor? weight, Tensor? bias, float eps"
#define XNN_DENSE_SCHEMA \
  "Tensor x, Tensor weight, Tensor? bias, int activation, Tensor? residual, Tensor? plan"

#define XNN_OPERATORS(X)                      \
  X(layer_norm, layer_norm)                   \
  X(layer_norm_stats, layer_norm_stats)       \
  X(layer_norm_backward, layer_norm_backward) \
  X(group_plan, group_plan)                   \
  X(dense, dense)                             \
  X(dense_slope, dense_slope)                 \
  X(dense_backward, dense_backward)

}  // namespace

TORCH_LIBRARY_FRAGMENT(xnn_amd, m) {
  m.def("layer_norm(" XNN_NORM_SCHEMA ") -> Tensor");
  m.def("layer_norm_stats(" XNN_NORM_SCHEMA ") -> (Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor stats, bool input, bool weights, "
        "bool biases) -> (Tensor, Tensor, Tensor)");
  m.def("group_plan(Tensor ids, int n_groups) -> Tensor");
  m.def("dense(" XNN_DENSE_SCHEMA ") -> Tensor");
  m.def("dense_slope(" XNN_DENSE_SCHEMA ") -> (Tensor, Tensor)");
  m.def("dense_backward(Tensor grad, Tensor? slope, Tensor? x, Tensor? weight, Tensor? plan, bool input, "
        "bool weights, bool biases) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(xnn_amd, CUDA, m) { XNN_OPERATORS(XNN_IMPL_KERNEL) }
// refused there by the same checks
TORCH_LIBRARY_IMPL(xnn_amd, CPU, m) { XNN_OPERATORS(XNN_IMPL_KERNEL) }
TORCH_LIBRARY_IMPL(xnn_amd, Meta, m) { XNN_OPERATORS(XNN_IMPL_SHAPE) }
TORCH_LIBRARY_IMPL(xnn_amd, FuncTorchBatched, m) { XNN_OPERATORS(XNN_IMPL_REFUSE) }
TORCH_LIBRARY_IMPL(xnn_amd, Autograd, m) {
  m.impl("layer_norm", &layer_norm_autograd);
  m.impl("dense", &dense_autograd);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_library", [](const std::string& path) { library = path; });
  m.def("entries", &entries);
  m.def("calls", &calls);
  m.def("layer_norm", &layer_norm);
  m.def("group_plan", &group_plan);
  m.def("dense", &dense);
}
