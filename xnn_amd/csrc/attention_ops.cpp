// The attention operators as operators of libtorch's dispatcher, with their autograd nodes, over the C ABI
// (host code).
//
// Their smallest calls are launches of a few microseconds: forward and backward run here without the
// interpreter, which costs 20 us a call in the forward pass and, on the thread of the backward pass, 40 more
// than these nodes. The library is opened by path and holds every kernel; nothing here computes.
//
// Each operator has a kernel for tensors with memory (checks, allocation, launch), one for shapes alone, and
// one that records its node; tracers, fake tensors and compilers see the operator, not the launch inside
// it. Checks raise ValueError, TypeError or, off the GPU, RuntimeError.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <atomic>
#include <limits>
#include <mutex>

#include "xnn_amd.h"

namespace {

using at::Tensor;
using torch::autograd::collect_next_edges;
using torch::autograd::deleteNode;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::set_history;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- the library
#define XNN_ENTRIES(X)                                                                         \
  X(xnn_last_error) X(xnn_embedding) X(xnn_embedding_grad_work_size) X(xnn_embedding_grad)     \
  X(xnn_dropout_add) X(xnn_head_norm_rotate) X(xnn_head_norm_rotate_backward_work_size)        \
  X(xnn_head_norm_rotate_backward) X(xnn_attention_work_size) X(xnn_attention)                 \
  X(xnn_attention_backward_work_size) X(xnn_attention_backward)

#define XNN_MEMBER(name) decltype(&::name) name = nullptr;
struct Api {
  XNN_ENTRIES(XNN_MEMBER)
} api;
#define XNN_COUNTER(name) std::atomic<int64_t> name{0};
struct Counts {
  XNN_ENTRIES(XNN_COUNTER)
} counts;

std::string library;

void open_library() {
  TORCH_CHECK(!library.empty(), "the path of the library is not set");
  void* lib = dlopen(library.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib != nullptr, dlerror());
#define XNN_RESOLVE(name)                                                \
  api.name = reinterpret_cast<decltype(&::name)>(dlsym(lib, #name));     \
  TORCH_CHECK(api.name != nullptr, library, " has no entry point " #name);
  XNN_ENTRIES(XNN_RESOLVE)
}

// opened by the first kernel that runs (a later one tries again where this failed)
void need_library() {
  static std::once_flag once;
  std::call_once(once, open_library);
}

int64_t calls(const std::string& name) {
#define XNN_COUNT(entry) \
  if (name == #entry) return counts.entry.load();
  XNN_ENTRIES(XNN_COUNT)
  return 0;
}

std::vector<std::string> entries() {
#define XNN_NAME(entry) #entry,
  return {XNN_ENTRIES(XNN_NAME)};
}

void check(const char* name, int status) {
  if (status == XNN_OK) return;
  TORCH_CHECK_VALUE(status != XNN_EINVAL, name, ": ", api.xnn_last_error());
  TORCH_CHECK(false, name, " failed: ", api.xnn_last_error());
}
#define XNN_CALL(name, ...)                  \
  do {                                       \
    ++counts.name;                           \
    check(#name, api.name(__VA_ARGS__));     \
  } while (0)

// ---------------------------------------------------------------- checks
int storage_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return XNN_F32;
    case at::kBFloat16: return XNN_BF16;
    case at::kHalf: return XNN_F16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(),
                              " (float32, bfloat16 or float16)");
  }
}

// every tensor on one GPU
void check_tensors(std::initializer_list<const Tensor*> ts) {
  need_library();
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "xnn_amd ops run on the GPU only (got a tensor on ", t->device(),
                "); there is no CPU fallback");
    TORCH_CHECK_VALUE(first == nullptr || t->device() == first->device(), "tensors on ", t->device(),
                      " and ", first->device());
    first = t;
  }
}

// none with a forward-mode tangent (which would be lost)
void refuse_tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(*t),
                                "the xnn_amd attention operators have no forward-mode derivative");
}

void check_integers(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(at::isIntegralType(t.scalar_type(), /*includeBool=*/false), name,
                   " must be integers, got ", t.scalar_type());
}

bool wanted(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void once_differentiable() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "the xnn_amd backward is differentiable once; double backward (create_graph=True) needs "
              "the PyTorch form (use_fast=False)");
}

xnn_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<xnn_stream_t>(
      c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream());
}

Tensor bytes(const Tensor& like, size_t n) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// an operator by its schema's name, with the signature of the function that names it here
#define XNN_OPERATOR(name, ...)                                                                \
  static const auto op =                                                                       \
      c10::Dispatcher::singleton().findSchemaOrThrow("xnn_amd::" name, "").typed<__VA_ARGS__>()

Tensor unit_stride(const Tensor& t) {
  return t.dim() != 3 || t.sym_stride(2) == 1 || t.sym_size(2) == 1 ? t : t.contiguous();
}

// integers as int64, anything else as it is (the kernel refuses it)
Tensor as_int64(const Tensor& t) {
  if (!t.defined() || !at::isIntegralType(t.scalar_type(), /*includeBool=*/false)) return t;
  return (t.scalar_type() == at::kLong ? t : t.to(at::kLong)).contiguous();
}

template <typename N, typename... Ts>
std::shared_ptr<N> node_of(const Ts&... inputs) {
  std::shared_ptr<N> node(new N(), deleteNode);
  node->set_next_edges(collect_next_edges(inputs...));
  return node;
}

// ---------------------------------------------------------------- embedding
Tensor embedding(const Tensor& ids, const Tensor& table, double scale) {
  XNN_OPERATOR("embedding_rows", Tensor(const Tensor&, const Tensor&, double));
  return op.call(ids, table, scale);
}

Tensor embedding_grad(const Tensor& ids, const Tensor& grad, c10::SymInt rows, double scale) {
  XNN_OPERATOR("embedding_rows_grad", Tensor(const Tensor&, const Tensor&, c10::SymInt, double));
  return op.call(ids, grad, rows, scale);
}

Tensor embedding_kernel(const Tensor& ids_, const Tensor& table_, double scale) {
  check_tensors({&table_, &ids_});
  TORCH_CHECK_VALUE(table_.dim() == 2, "table must be (rows, channels), got ", table_.sizes());
  check_integers(ids_, "ids");
  const int code = storage_code(table_);
  const c10::DeviceGuard guard(table_.device());
  const Tensor ids = as_int64(ids_), table = table_.contiguous();
  auto sizes = ids.sizes().vec();
  sizes.push_back(table.size(1));
  Tensor out = at::empty(sizes, table.options());
  XNN_CALL(xnn_embedding, code, ids.const_data_ptr<int64_t>(), ids.numel(), data(table), table.size(0),
           table.size(1), (float)scale, data(out), stream_of(table));
  return out;
}

Tensor embedding_shape(const Tensor& ids, const Tensor& table, double) {
  auto sizes = ids.sym_sizes().vec();
  sizes.push_back(table.sym_size(1));
  return at::empty_symint(sizes, table.options());
}

Tensor embedding_grad_kernel(const Tensor& ids_, const Tensor& grad_, c10::SymInt rows_, double scale) {
  check_tensors({&grad_, &ids_});
  check_integers(ids_, "ids");
  const int code = storage_code(grad_);
  const c10::DeviceGuard guard(grad_.device());
  const Tensor ids = as_int64(ids_), grad = grad_.contiguous();
  const int64_t rows = rows_.expect_int();
  TORCH_CHECK_VALUE(rows >= 0 && grad.dim() == ids.dim() + 1 &&
                        grad.sizes().slice(0, ids.dim()) == ids.sizes(),
                    "a cotangent ", grad.sizes(), " of ids ", ids.sizes());
  const int64_t channels = grad.size(-1);
  Tensor out = at::empty({rows, channels}, grad.options());
  size_t need = 0;
  check("xnn_embedding_grad_work_size",
        api.xnn_embedding_grad_work_size(ids.numel(), rows, channels, &need));
  const Tensor work = bytes(grad, need);
  XNN_CALL(xnn_embedding_grad, code, ids.const_data_ptr<int64_t>(), ids.numel(), data(grad), rows, channels,
           (float)scale, data(out), data(work), need, stream_of(grad));
  return out;
}

Tensor embedding_grad_shape(const Tensor&, const Tensor& grad, c10::SymInt rows, double) {
  return at::empty_symint({rows, grad.sym_size(-1)}, grad.options());
}

struct EmbeddingBackward : Node {
  SavedVariable ids;
  c10::SymInt rows;
  double scale;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    return {embedding_grad(ids.unpack(), grads[0], rows, scale)};
  }
  void release_variables() override { ids.reset_data(); }
  std::string name() const override { return "XnnEmbeddingBackward"; }
};

// the two are each other's adjoints: differentiable to any order
struct EmbeddingGradBackward : Node {
  SavedVariable ids;
  double scale;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    return {embedding(ids.unpack(), grads[0], scale)};
  }
  void release_variables() override { ids.reset_data(); }
  std::string name() const override { return "XnnEmbeddingGradBackward"; }
};

Tensor embedding_autograd(const Tensor& ids_, const Tensor& table, double scale) {
  refuse_tangents({&table});
  const bool train = wanted({&table});
  const Tensor ids = train ? as_int64(ids_) : ids_;
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = embedding(ids, table, scale);
  }
  if (train) {
    auto node = node_of<EmbeddingBackward>(table);
    node->ids = SavedVariable(ids, false);
    node->rows = table.sym_size(0);
    node->scale = scale;
    set_history(out, node);
  }
  return out;
}

Tensor embedding_grad_autograd(const Tensor& ids, const Tensor& grad, c10::SymInt rows, double scale) {
  refuse_tangents({&grad});
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = embedding_grad(ids, grad, rows, scale);
  }
  if (wanted({&grad})) {
    auto node = node_of<EmbeddingGradBackward>(grad);
    node->ids = SavedVariable(ids, false);
    node->scale = scale;
    set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------- dropout
typedef std::optional<Tensor> MaybeTensor;

Tensor dropout(const Tensor& x, const MaybeTensor& residual, double p, int64_t seed, int64_t offset,
               const MaybeTensor& counter) {
  XNN_OPERATOR("dropout_add",
               Tensor(const Tensor&, const MaybeTensor&, double, int64_t, int64_t, const MaybeTensor&));
  return op.call(x, residual, p, seed, offset, counter);
}

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

Tensor dropout_kernel(const Tensor& x_, const MaybeTensor& residual_, double p, int64_t seed, int64_t offset,
                      const MaybeTensor& counter_) {
  Tensor residual = or_none(residual_);
  const Tensor counter = or_none(counter_);
  check_tensors({&x_, &residual, &counter});
  const int code = storage_code(x_);
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == x_.sizes() &&
                                            residual.scalar_type() == x_.scalar_type()),
                    "residual ", residual.defined() ? residual.sizes() : x_.sizes(),
                    " does not match x ", x_.sizes(), " (sizes and dtype)");
  TORCH_CHECK_VALUE(!counter.defined() || (counter.scalar_type() == at::kLong && counter.numel() == 1),
                    "an offset tensor holds one int64");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = x_.contiguous();
  if (residual.defined()) residual = residual.contiguous();
  Tensor out = at::empty(x.sizes(), x.options());
  XNN_CALL(xnn_dropout_add, code, data(x), data(residual), x.numel(), (int32_t)std::nearbyint(p * 65536),
           (uint64_t)seed, (uint64_t)offset, (const int64_t*)data(counter), data(out), stream_of(x));
  return out;
}

Tensor dropout_shape(const Tensor& x, const MaybeTensor&, double, int64_t, int64_t, const MaybeTensor&) {
  return at::empty_symint(x.sym_sizes(), x.options());
}

struct DropoutBackward : Node {
  SavedVariable counter;
  double p;
  int64_t seed, offset;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    Tensor dx;
    if (task_should_compute_output(0))
      dx = dropout(grads[0], MaybeTensor(), p, seed, offset, maybe(counter.unpack()));
    return {dx, task_should_compute_output(1) ? grads[0] : Tensor()};
  }
  void release_variables() override { counter.reset_data(); }
  std::string name() const override { return "XnnDropoutBackward"; }
};

Tensor dropout_autograd(const Tensor& x, const MaybeTensor& residual_, double p, int64_t seed, int64_t offset,
                        const MaybeTensor& counter) {
  const Tensor residual = or_none(residual_), c = or_none(counter);
  refuse_tangents({&x, &residual});
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = dropout(x, residual_, p, seed, offset, counter);
  }
  if (wanted({&x, &residual})) {
    auto node = node_of<DropoutBackward>(x, residual);
    node->counter = SavedVariable(c, false);
    node->p = p;
    node->seed = seed;
    node->offset = offset;
    set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------- norm and rotation
typedef std::tuple<Tensor, Tensor> Two;

xnn_heads heads_of(const Tensor& t) {
  return xnn_heads{t.data_ptr(), t.stride(0), t.stride(1), (int32_t)t.size(1)};
}

constexpr int64_t kMaxHeadDim = 128;

Two head_norm_rotate(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                     const Tensor& cos, const Tensor& sin, const MaybeTensor& positions, double eps,
                     bool interleaved) {
  XNN_OPERATOR("head_norm_rotate",
               Two(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                   const MaybeTensor&, double, bool));
  return op.call(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
}

// the gradients of q, k, their weights, cos and sin; without `weights` or `tables` theirs are empty
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Six;

Six head_norm_rotate_backward(const Tensor& grad_q, const Tensor& grad_k, const Tensor& q, const Tensor& k,
                              const Tensor& q_weight, const Tensor& k_weight, const Tensor& cos,
                              const Tensor& sin, const MaybeTensor& positions, double eps, bool interleaved,
                              bool weights, bool tables) {
  XNN_OPERATOR("head_norm_rotate_backward",
               Six(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                   const Tensor&, const Tensor&, const MaybeTensor&, double, bool, bool, bool));
  return op.call(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, weights,
                 tables);
}

void check_heads(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                 const Tensor& cos, const Tensor& sin, const Tensor& positions) {
  check_tensors({&q, &k, &q_weight, &k_weight, &cos, &sin, &positions});
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                    "q and k must be (tokens, heads, head_dim) of the same tokens and head_dim, got ",
                    q.sizes(), " and ", k.sizes());
  const int64_t T = q.size(0), D = q.size(2);
  TORCH_CHECK_VALUE(D >= 1 && D <= kMaxHeadDim, "head_dim must be in [1, ", kMaxHeadDim, "], got ", D);
  TORCH_CHECK_VALUE(q.size(1) >= 1 && k.size(1) >= 1, "no heads");
  storage_code(q);
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && q_weight.scalar_type() == q.scalar_type() &&
                       k_weight.scalar_type() == q.scalar_type(),
                   "q, k and their weights must have one dtype");
  TORCH_CHECK_VALUE(q_weight.dim() == 1 && q_weight.size(0) == D && k_weight.dim() == 1 &&
                        k_weight.size(0) == D,
                    "the weights must be (", D, ",)");
  TORCH_CHECK_TYPE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
                   "cos and sin must be float32");
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && 2 * cos.size(1) <= D,
                    "cos and sin must be (rows, R / 2) with R <= ", D, ", got ", cos.sizes(), " and ",
                    sin.sizes());
  if (!positions.defined()) {
    TORCH_CHECK_VALUE(cos.size(0) == T, "without positions the tables have a row a token: ", cos.size(0),
                      " rows, ", T, " tokens");
  } else {
    TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == T &&
                          at::isIntegralType(positions.scalar_type(), false),
                      "positions must be (", T, ",) integers");
  }
}

Two head_norm_rotate_kernel(const Tensor& q_, const Tensor& k_, const Tensor& q_weight_,
                            const Tensor& k_weight_, const Tensor& cos_, const Tensor& sin_,
                            const MaybeTensor& positions_, double eps, bool interleaved) {
  check_heads(q_, k_, q_weight_, k_weight_, cos_, sin_, or_none(positions_));
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = unit_stride(q_), k = unit_stride(k_), q_weight = q_weight_.contiguous(),
               k_weight = k_weight_.contiguous(), cos = cos_.contiguous(), sin = sin_.contiguous(),
               positions = as_int64(or_none(positions_));
  Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
  const xnn_heads qh = heads_of(q), kh = heads_of(k);
  XNN_CALL(xnn_head_norm_rotate, storage_code(q), &qh, &kh, q.size(0), (int32_t)q.size(2),
           (int32_t)(2 * cos.size(1)), data(q_weight), data(k_weight), cos.const_data_ptr<float>(),
           sin.const_data_ptr<float>(), cos.size(0), (const int64_t*)data(positions), (float)eps, interleaved,
           data(q_out), data(k_out), stream_of(q));
  return {q_out, k_out};
}

Two head_norm_rotate_shape(const Tensor& q, const Tensor& k, const Tensor&, const Tensor&, const Tensor&,
                           const Tensor&, const MaybeTensor&, double, bool) {
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}

Six head_norm_rotate_backward_kernel(const Tensor& grad_q, const Tensor& grad_k, const Tensor& q_,
                                     const Tensor& k_, const Tensor& q_weight_, const Tensor& k_weight_,
                                     const Tensor& cos_, const Tensor& sin_, const MaybeTensor& positions_,
                                     double eps, bool interleaved, bool weights, bool tables) {
  check_heads(q_, k_, q_weight_, k_weight_, cos_, sin_, or_none(positions_));
  check_tensors({&q_, &grad_q, &grad_k});
  TORCH_CHECK_VALUE(grad_q.sizes() == q_.sizes() && grad_k.sizes() == k_.sizes() &&
                        grad_q.scalar_type() == q_.scalar_type() && grad_k.scalar_type() == k_.scalar_type(),
                    "cotangents ", grad_q.sizes(), " and ", grad_k.sizes(), " of ", q_.sizes(), " and ",
                    k_.sizes(), " (sizes and dtype)");
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = unit_stride(q_), k = unit_stride(k_), q_weight = q_weight_.contiguous(),
               k_weight = k_weight_.contiguous(), cos = cos_.contiguous(), sin = sin_.contiguous(),
               positions = as_int64(or_none(positions_)), gq = grad_q.contiguous(), gk = grad_k.contiguous();
  const auto like = [](const Tensor& t, bool wanted) {
    return wanted ? at::empty(t.sizes(), t.options()) : at::empty({0}, t.options());
  };
  const Tensor dq = like(q, true), dk = like(k, true), dqw = like(q_weight, weights),
               dkw = like(k_weight, weights), dc = like(cos, tables), ds = like(sin, tables);
  Tensor work;
  size_t need = 0;
  if (weights) {
    check("xnn_head_norm_rotate_backward_work_size",
          api.xnn_head_norm_rotate_backward_work_size((int32_t)q.size(2), &need));
    work = bytes(q, need);
  }
  const xnn_heads qh = heads_of(q), kh = heads_of(k);
  XNN_CALL(xnn_head_norm_rotate_backward, storage_code(q), &qh, &kh, q.size(0), (int32_t)q.size(2),
           (int32_t)(2 * cos.size(1)), data(q_weight), data(k_weight), cos.const_data_ptr<float>(),
           sin.const_data_ptr<float>(), cos.size(0), (const int64_t*)data(positions), (float)eps, interleaved,
           data(gq), data(gk), data(dq), data(dk), data(dqw), data(dkw), (float*)data(dc),
           (float*)data(ds), data(work), need, stream_of(q));
  return {dq, dk, dqw, dkw, dc, ds};
}

Six head_norm_rotate_backward_shape(const Tensor&, const Tensor&, const Tensor& q, const Tensor& k,
                                    const Tensor& q_weight, const Tensor& k_weight, const Tensor& cos,
                                    const Tensor& sin, const MaybeTensor&, double, bool, bool weights,
                                    bool tables) {
  const auto like = [](const Tensor& t, bool wanted) {
    return wanted ? at::empty_symint(t.sym_sizes(), t.options()) : at::empty({0}, t.options());
  };
  return {like(q, true),          like(k, true),     like(q_weight, weights),
          like(k_weight, weights), like(cos, tables), like(sin, tables)};
}

struct NormRotateBackward : Node {
  SavedVariable q, k, q_weight, k_weight, cos, sin, positions;
  double eps;
  bool interleaved;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable();
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const Tensor q = this->q.unpack(), k = this->k.unpack(), qw = q_weight.unpack(), kw = k_weight.unpack(),
                 c = cos.unpack(), s = sin.unpack(), pos = positions.unpack();
    const bool weights = task_should_compute_output(2) || task_should_compute_output(3);
    const bool tables = task_should_compute_output(4) || task_should_compute_output(5);
    at::AutoDispatchBelowADInplaceOrView below;            // no derivative of its own
    const Tensor gq = grads[0].defined() ? grads[0] : at::zeros_symint(q.sym_sizes(), q.options());
    const Tensor gk = grads[1].defined() ? grads[1] : at::zeros_symint(k.sym_sizes(), k.options());
    const Six all = head_norm_rotate_backward(gq, gk, q, k, qw, kw, c, s, maybe(pos), eps, interleaved, weights,
                                              tables);
    const auto& [dq, dk, dqw, dkw, dc, ds] = all;
    const Tensor* each[] = {&dq, &dk, &dqw, &dkw, &dc, &ds};
    for (int i = 0; i < 6; ++i)
      if (task_should_compute_output(i)) out[i] = *each[i];
    return out;
  }
  void release_variables() override {
    for (SavedVariable* v : {&q, &k, &q_weight, &k_weight, &cos, &sin, &positions}) v->reset_data();
  }
  std::string name() const override { return "XnnHeadNormRotateBackward"; }
};

Two head_norm_rotate_autograd(const Tensor& q_, const Tensor& k_, const Tensor& q_weight_,
                              const Tensor& k_weight_, const Tensor& cos_, const Tensor& sin_,
                              const MaybeTensor& positions_, double eps, bool interleaved) {
  refuse_tangents({&q_, &k_, &q_weight_, &k_weight_, &cos_, &sin_});
  const bool train = wanted({&q_, &k_, &q_weight_, &k_weight_, &cos_, &sin_});
  if (!train) {
    at::AutoDispatchBelowADInplaceOrView below;
    return head_norm_rotate(q_, k_, q_weight_, k_weight_, cos_, sin_, positions_, eps, interleaved);
  }
  const Tensor positions = as_int64(or_none(positions_));
  TORCH_CHECK_VALUE(!positions.defined() || !wanted({&cos_, &sin_}),
                    "tables read by position have no gradient here (gather their rows and leave positions "
                    "out)");
  const Tensor q = unit_stride(q_), k = unit_stride(k_), q_weight = q_weight_.contiguous(),
               k_weight = k_weight_.contiguous(), cos = cos_.contiguous(), sin = sin_.contiguous();
  Two out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = head_norm_rotate(q, k, q_weight, k_weight, cos, sin, maybe(positions), eps, interleaved);
  }
  auto node = node_of<NormRotateBackward>(q, k, q_weight, k_weight, cos, sin);
  node->q = SavedVariable(q, false);
  node->k = SavedVariable(k, false);
  node->q_weight = SavedVariable(q_weight, false);
  node->k_weight = SavedVariable(k_weight, false);
  node->cos = SavedVariable(cos, false);
  node->sin = SavedVariable(sin, false);
  node->positions = SavedVariable(positions, false);
  node->eps = eps;
  node->interleaved = interleaved;
  set_history(std::get<0>(out), node);
  set_history(std::get<1>(out), node);
  return out;
}

// ---------------------------------------------------------------- attention
typedef std::tuple<Tensor, Tensor, Tensor> Three;

// a plan as the kernels take it
struct Tiles {
  Tensor tiles32, tiles128;
  xnn_attention_tiles c;
  Tiles(const Tensor& tiles32_, const Tensor& tiles128_, const c10::SymInt& n_tokens,
        const c10::SymInt& max_atoms) {
    for (const Tensor* t : {&tiles32_, &tiles128_})
      TORCH_CHECK_VALUE(t->dim() == 2 && t->size(1) == 3 && t->scalar_type() == at::kInt,
                        "a plan's tiles are (n, 3) int32, got ", t->sizes(), " ", t->scalar_type());
    tiles32 = tiles32_.contiguous();
    tiles128 = tiles128_.contiguous();
    c = xnn_attention_tiles{n_tokens.expect_int(), max_atoms.expect_int(),         tiles32.size(0),
                            tiles128.size(0),      (const int32_t*)data(tiles32),  (const int32_t*)data(tiles128)};
  }
};

#define XNN_ATTENTION_ARGUMENTS                                                                         \
  const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &tiles32, const Tensor &tiles128,     \
      const MaybeTensor &mask, c10::SymInt n_tokens, c10::SymInt max_atoms, std::optional<double> scale
#define XNN_ATTENTION_TYPES                                                                             \
  const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const MaybeTensor&,        \
      c10::SymInt, c10::SymInt, std::optional<double>

Tensor structure_attention(XNN_ATTENTION_ARGUMENTS) {
  XNN_OPERATOR("structure_attention", Tensor(XNN_ATTENTION_TYPES));
  return op.call(q, k, v, tiles32, tiles128, mask, n_tokens, max_atoms, scale);
}

// with the rows' log-sums
Two structure_attention_lse(XNN_ATTENTION_ARGUMENTS) {
  XNN_OPERATOR("structure_attention_lse", Two(XNN_ATTENTION_TYPES));
  return op.call(q, k, v, tiles32, tiles128, mask, n_tokens, max_atoms, scale);
}

Three structure_attention_backward(const Tensor& grad, const Tensor& out, const Tensor& lse,
                                   XNN_ATTENTION_ARGUMENTS) {
  XNN_OPERATOR("structure_attention_backward",
               Three(const Tensor&, const Tensor&, const Tensor&, XNN_ATTENTION_TYPES));
  return op.call(grad, out, lse, q, k, v, tiles32, tiles128, mask, n_tokens, max_atoms, scale);
}

double check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tiles& plan, const Tensor& mask,
                       const std::optional<double>& scale_) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
                        q.size(2) == k.size(2),
                    "q must be (tokens, heads, head_dim), k and v (tokens, kv_heads, head_dim), got ",
                    q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK_VALUE(D >= 1 && D <= kMaxHeadDim, "head_dim must be in [1, ", kMaxHeadDim, "], got ", D);
  TORCH_CHECK_VALUE(k.size(1) >= 1 && H >= 1 && H % k.size(1) == 0, H, " heads cannot share ", k.size(1),
                    " heads of keys and values");
  storage_code(q);
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k and v must have one dtype, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(plan.c.n_tokens == T, "the plan is of ", plan.c.n_tokens, " tokens, q holds ", T);
  TORCH_CHECK_VALUE(!mask.defined() || (mask.dim() == 1 && mask.size(0) == T && mask.scalar_type() == at::kBool),
                    "mask must be (", T, ",) bool, got ", mask.defined() ? mask.sizes() : q.sizes());
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(scale > 0.0 && scale < std::numeric_limits<double>::infinity(),
                    "scale must be positive and finite, got ", scale);
  return scale;
}

Two attention_forward(XNN_ATTENTION_ARGUMENTS, bool keep) {
  Tensor m = or_none(mask);
  check_tensors({&q, &k, &v, &m, &tiles32, &tiles128});
  const c10::DeviceGuard guard(q.device());
  const Tiles plan(tiles32, tiles128, n_tokens, max_atoms);
  const double s = check_attention(q, k, v, plan, m, scale);
  if (m.defined()) m = m.contiguous();
  const Tensor a = unit_stride(q), b = unit_stride(k), c = unit_stride(v);
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  const int code = storage_code(q);
  Tensor out = at::empty(q.sizes(), q.options()), lse, work;
  if (keep) lse = at::empty({H, T}, q.options().dtype(at::kFloat));
  size_t need = 0;
  check("xnn_attention_work_size",
        api.xnn_attention_work_size(code, T, (int32_t)H, (int32_t)D, &plan.c, &need));
  if (need > 0) work = bytes(q, need);
  const xnn_heads qh = heads_of(a), kh = heads_of(b), vh = heads_of(c);
  XNN_CALL(xnn_attention, code, &qh, &kh, &vh, T, (int32_t)D, &plan.c, (const uint8_t*)data(m), (float)s,
           data(out), (float*)data(lse), data(work), need, stream_of(q));
  return {out, lse};
}

Tensor structure_attention_kernel(XNN_ATTENTION_ARGUMENTS) {
  return std::get<0>(attention_forward(q, k, v, tiles32, tiles128, mask, n_tokens, max_atoms, scale, false));
}
Two structure_attention_lse_kernel(XNN_ATTENTION_ARGUMENTS) {
  return attention_forward(q, k, v, tiles32, tiles128, mask, n_tokens, max_atoms, scale, true);
}

Tensor structure_attention_shape(XNN_ATTENTION_ARGUMENTS) {
  return at::empty_symint(q.sym_sizes(), q.options());
}
Two structure_attention_lse_shape(XNN_ATTENTION_ARGUMENTS) {
  return {at::empty_symint(q.sym_sizes(), q.options()),
          at::empty_symint({q.sym_size(1), q.sym_size(0)}, q.options().dtype(at::kFloat))};
}

Three structure_attention_backward_kernel(const Tensor& grad, const Tensor& out, const Tensor& lse,
                                          XNN_ATTENTION_ARGUMENTS) {
  Tensor m = or_none(mask);
  check_tensors({&q, &k, &v, &m, &tiles32, &tiles128, &grad, &out, &lse});
  const c10::DeviceGuard guard(q.device());
  const Tiles plan(tiles32, tiles128, n_tokens, max_atoms);
  const double s = check_attention(q, k, v, plan, m, scale);
  TORCH_CHECK_VALUE(grad.sizes() == q.sizes() && out.sizes() == q.sizes() &&
                        grad.scalar_type() == q.scalar_type() && out.scalar_type() == q.scalar_type(),
                    "a cotangent ", grad.sizes(), " and an output ", out.sizes(), " of ", q.sizes(),
                    " (sizes and dtype)");
  TORCH_CHECK_VALUE(lse.dim() == 2 && lse.size(0) == q.size(1) && lse.size(1) == q.size(0) &&
                        lse.scalar_type() == at::kFloat,
                    "log-sums ", lse.sizes(), " of q ", q.sizes());
  if (m.defined()) m = m.contiguous();
  const Tensor a = unit_stride(q), b = unit_stride(k), c = unit_stride(v), g = grad.contiguous(),
               o = out.contiguous(), l = lse.contiguous();
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
         dv = at::empty(v.sizes(), v.options());
  const int code = storage_code(q);
  size_t need = 0;
  check("xnn_attention_backward_work_size",
        api.xnn_attention_backward_work_size(code, q.size(0), (int32_t)q.size(1), (int32_t)k.size(1),
                                             (int32_t)q.size(2), &plan.c, &need));
  const Tensor work = bytes(q, need);
  const xnn_heads qh = heads_of(a), kh = heads_of(b), vh = heads_of(c);
  XNN_CALL(xnn_attention_backward, code, &qh, &kh, &vh, q.size(0), (int32_t)q.size(2), &plan.c,
           (const uint8_t*)data(m), (float)s, data(o), l.const_data_ptr<float>(), data(g), data(dq), data(dk),
           data(dv), data(work), need, stream_of(q));
  return {dq, dk, dv};
}

Three structure_attention_backward_shape(const Tensor&, const Tensor&, const Tensor&, XNN_ATTENTION_ARGUMENTS) {
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options()),
          at::empty_symint(v.sym_sizes(), v.options())};
}

struct AttentionBackward : Node {
  SavedVariable q, k, v, mask, out, lse, tiles32, tiles128;
  c10::SymInt n_tokens, max_atoms;
  std::optional<double> scale;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable();
    variable_list result(3);
    if (!grads[0].defined()) return result;
    at::AutoDispatchBelowADInplaceOrView below;            // no derivative of its own
    const Three all = structure_attention_backward(
        grads[0], out.unpack(shared_from_this()), lse.unpack(), q.unpack(), k.unpack(), v.unpack(),
        tiles32.unpack(), tiles128.unpack(), maybe(mask.unpack()), n_tokens, max_atoms, scale);
    if (task_should_compute_output(0)) result[0] = std::get<0>(all);
    if (task_should_compute_output(1)) result[1] = std::get<1>(all);
    if (task_should_compute_output(2)) result[2] = std::get<2>(all);
    return result;
  }
  void release_variables() override {
    for (SavedVariable* s : {&q, &k, &v, &mask, &out, &lse, &tiles32, &tiles128}) s->reset_data();
  }
  std::string name() const override { return "XnnAttentionBackward"; }
};

Tensor structure_attention_autograd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& tiles32,
                                    const Tensor& tiles128, const MaybeTensor& mask_, c10::SymInt n_tokens,
                                    c10::SymInt max_atoms, std::optional<double> scale) {
  refuse_tangents({&q_, &k_, &v_});
  if (!wanted({&q_, &k_, &v_})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return structure_attention(q_, k_, v_, tiles32, tiles128, mask_, n_tokens, max_atoms, scale);
  }
  const Tensor q = unit_stride(q_), k = unit_stride(k_), v = unit_stride(v_);
  Tensor mask = or_none(mask_), out, lse;
  if (mask.defined()) mask = mask.contiguous();
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(out, lse) =
        structure_attention_lse(q, k, v, tiles32, tiles128, maybe(mask), n_tokens, max_atoms, scale);
  }
  auto node = node_of<AttentionBackward>(q, k, v);
  node->q = SavedVariable(q, false);
  node->k = SavedVariable(k, false);
  node->v = SavedVariable(v, false);
  node->mask = SavedVariable(mask, false);
  node->lse = SavedVariable(lse, false);
  node->tiles32 = SavedVariable(tiles32, false);
  node->tiles128 = SavedVariable(tiles128, false);
  node->n_tokens = n_tokens;
  node->max_atoms = max_atoms;
  node->scale = scale;
  set_history(out, node);
  node->out = SavedVariable(out, true);
  return out;
}

// ---------------------------------------------------------------- registration
// No rule for a batch of calls: a loop over them would draw one dropout mask for all. (A batch of cotangents
// is such a loop over the backward operators.)
void refuse_batches(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().name(), " has no batching rule (vmap)");
}

#define XNN_ATTENTION_SCHEMA                                                                       \
  "Tensor q, Tensor k, Tensor v, Tensor tiles32, Tensor tiles128, Tensor? mask, SymInt n_tokens, " \
  "SymInt max_atoms, float? scale"
#define XNN_HEADS_SCHEMA                                                                          \
  "Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, Tensor sin, Tensor? positions, " \
  "float eps, bool interleaved"

#define XNN_OPERATORS(X)                                                                            \
  X(embedding_rows, embedding)                                                                      \
  X(embedding_rows_grad, embedding_grad)                                                            \
  X(dropout_add, dropout)                                                                           \
  X(head_norm_rotate, head_norm_rotate)                                                             \
  X(head_norm_rotate_backward, head_norm_rotate_backward)                                           \
  X(structure_attention, structure_attention)                                                       \
  X(structure_attention_lse, structure_attention_lse)                                               \
  X(structure_attention_backward, structure_attention_backward)

}  // namespace

TORCH_LIBRARY_FRAGMENT(xnn_amd, m) {
  m.def("embedding_rows(Tensor ids, Tensor table, float scale) -> Tensor");
  m.def("embedding_rows_grad(Tensor ids, Tensor grad, SymInt rows, float scale) -> Tensor");
  m.def("dropout_add(Tensor x, Tensor? residual, float p, int seed, int offset, Tensor? counter) -> Tensor");
  m.def("head_norm_rotate(" XNN_HEADS_SCHEMA ") -> (Tensor, Tensor)");
  m.def("head_norm_rotate_backward(Tensor grad_q, Tensor grad_k, " XNN_HEADS_SCHEMA
        ", bool weights, bool tables) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("structure_attention(" XNN_ATTENTION_SCHEMA ") -> Tensor");
  m.def("structure_attention_lse(" XNN_ATTENTION_SCHEMA ") -> (Tensor, Tensor)");
  m.def("structure_attention_backward(Tensor grad, Tensor out, Tensor lse, " XNN_ATTENTION_SCHEMA
        ") -> (Tensor, Tensor, Tensor)");
}

#define XNN_IMPL_KERNEL(schema, f) m.impl(#schema, &f##_kernel);
#define XNN_IMPL_SHAPE(schema, f) m.impl(#schema, &f##_shape);
#define XNN_IMPL_REFUSE(schema, f) \
  m.impl(#schema, torch::CppFunction::makeFromBoxedFunction<&refuse_batches>());

TORCH_LIBRARY_IMPL(xnn_amd, CUDA, m) { XNN_OPERATORS(XNN_IMPL_KERNEL) }
// refused there by the same checks
TORCH_LIBRARY_IMPL(xnn_amd, CPU, m) { XNN_OPERATORS(XNN_IMPL_KERNEL) }
TORCH_LIBRARY_IMPL(xnn_amd, Meta, m) { XNN_OPERATORS(XNN_IMPL_SHAPE) }
TORCH_LIBRARY_IMPL(xnn_amd, FuncTorchBatched, m) { XNN_OPERATORS(XNN_IMPL_REFUSE) }
TORCH_LIBRARY_IMPL(xnn_amd, Autograd, m) {
  m.impl("embedding_rows", &embedding_autograd);
  m.impl("embedding_rows_grad", &embedding_grad_autograd);
  m.impl("dropout_add", &dropout_autograd);
  m.impl("head_norm_rotate", &head_norm_rotate_autograd);
  m.impl("structure_attention", &structure_attention_autograd);
}

namespace {

Tensor dropout_entry(const Tensor& x, const MaybeTensor& residual, double p, uint64_t seed, uint64_t offset,
                     const MaybeTensor& counter) {
  return dropout(x, residual, p, (int64_t)seed, (int64_t)offset, counter);
}

struct Plan {
  c10::SymInt n_tokens, max_atoms;
  Tensor tiles32, tiles128;
};

Tensor structure_attention_entry(const Tensor& q, const Tensor& k, const Tensor& v, const Plan& plan,
                                 const MaybeTensor& mask, const std::optional<double>& scale) {
  return structure_attention(q, k, v, plan.tiles32, plan.tiles128, mask, plan.n_tokens, plan.max_atoms, scale);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("set_library", [](const std::string& path) { library = path; });
  m.def("entries", &entries);
  m.def("calls", &calls);
  m.def("embedding", &embedding);
  m.def("dropout_add", &dropout_entry);
  m.def("head_norm_rotate", &head_norm_rotate);
  m.def("structure_attention", &structure_attention_entry);
  py::class_<Plan>(m, "Plan").def(py::init([](int64_t n_tokens, int64_t max_atoms, const Tensor& tiles32,
                                              const Tensor& tiles128) {
    return Plan{n_tokens, max_atoms, tiles32, tiles128};
  }));
}
