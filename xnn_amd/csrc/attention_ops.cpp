// The attention operators as autograd functions of libtorch, over the C ABI (host code).
//
// Their smallest calls are launches of a few microseconds: forward and backward run here without the
// interpreter, which costs 20 us a call in the forward pass and, on the thread of the backward pass, 40 more
// than these nodes. The library is opened by path and holds every kernel; nothing here computes.
// Checks raise ValueError, TypeError or, off the GPU, RuntimeError.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

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

void load(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib != nullptr, dlerror());
#define XNN_RESOLVE(name)                                                \
  api.name = reinterpret_cast<decltype(&::name)>(dlsym(lib, #name));     \
  TORCH_CHECK(api.name != nullptr, path, " has no entry point " #name);
  XNN_ENTRIES(XNN_RESOLVE)
}

int64_t calls(const std::string& name) {
#define XNN_COUNT(entry) \
  if (name == #entry) return counts.entry.load();
  XNN_ENTRIES(XNN_COUNT)
  return 0;
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

// every tensor on one GPU, none with a forward-mode tangent (which would be lost)
void check_tensors(std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "xnn_amd ops run on the GPU only (got a tensor on ", t->device(),
                "); there is no CPU fallback");
    TORCH_CHECK_VALUE(first == nullptr || t->device() == first->device(), "tensors on ", t->device(),
                      " and ", first->device());
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(*t),
                                "the xnn_amd attention operators have no forward-mode derivative");
    first = t;
  }
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

template <typename N, typename... Ts>
std::shared_ptr<N> node_of(const Ts&... inputs) {
  std::shared_ptr<N> node(new N(), deleteNode);
  node->set_next_edges(collect_next_edges(inputs...));
  return node;
}

// ---------------------------------------------------------------- embedding
Tensor embedding(Tensor ids, Tensor table, double scale);
Tensor embedding_grad(const Tensor& ids, Tensor grad, int64_t rows, double scale);

struct EmbeddingBackward : Node {
  SavedVariable ids;
  int64_t rows;
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

Tensor embedding(Tensor ids, Tensor table, double scale) {
  check_tensors({&table, &ids});
  TORCH_CHECK_VALUE(table.dim() == 2, "table must be (rows, channels), got ", table.sizes());
  check_integers(ids, "ids");
  const int code = storage_code(table);
  const c10::DeviceGuard guard(table.device());
  ids = ids.to(at::kLong).contiguous();
  table = table.contiguous();
  auto sizes = ids.sizes().vec();
  sizes.push_back(table.size(1));
  Tensor out = at::empty(sizes, table.options());
  XNN_CALL(xnn_embedding, code, ids.const_data_ptr<int64_t>(), ids.numel(), data(table), table.size(0),
           table.size(1), (float)scale, data(out), stream_of(table));
  if (wanted({&table})) {
    auto node = node_of<EmbeddingBackward>(table);
    node->ids = SavedVariable(ids, false);
    node->rows = table.size(0);
    node->scale = scale;
    set_history(out, node);
  }
  return out;
}

Tensor embedding_grad(const Tensor& ids, Tensor grad, int64_t rows, double scale) {
  const c10::DeviceGuard guard(grad.device());
  grad = grad.contiguous();
  const int64_t channels = grad.size(-1);
  Tensor out = at::empty({rows, channels}, grad.options());
  size_t need = 0;
  check("xnn_embedding_grad_work_size",
        api.xnn_embedding_grad_work_size(ids.numel(), rows, channels, &need));
  const Tensor work = bytes(grad, need);
  XNN_CALL(xnn_embedding_grad, storage_code(grad), ids.const_data_ptr<int64_t>(), ids.numel(), data(grad),
           rows, channels, (float)scale, data(out), data(work), need, stream_of(grad));
  if (wanted({&grad})) {
    auto node = node_of<EmbeddingGradBackward>(grad);
    node->ids = SavedVariable(ids, false);
    node->scale = scale;
    set_history(out, node);
  }
  return out;
}

// ---------------------------------------------------------------- dropout
Tensor dropout(Tensor x, Tensor residual, int64_t drop, uint64_t seed, uint64_t offset,
               const Tensor& counter);

struct DropoutBackward : Node {
  SavedVariable counter;
  int64_t drop;
  uint64_t seed, offset;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    Tensor dx;
    if (task_should_compute_output(0))
      dx = dropout(grads[0], Tensor(), drop, seed, offset, counter.unpack());
    return {dx, task_should_compute_output(1) ? grads[0] : Tensor()};
  }
  void release_variables() override { counter.reset_data(); }
  std::string name() const override { return "XnnDropoutBackward"; }
};

Tensor dropout(Tensor x, Tensor residual, int64_t drop, uint64_t seed, uint64_t offset,
               const Tensor& counter) {
  const c10::DeviceGuard guard(x.device());
  x = x.contiguous();
  if (residual.defined()) residual = residual.contiguous();
  Tensor out = at::empty(x.sizes(), x.options());
  XNN_CALL(xnn_dropout_add, storage_code(x), data(x), data(residual), x.numel(), (int32_t)drop, seed, offset,
           (const int64_t*)data(counter), data(out), stream_of(x));
  if (wanted({&x, &residual})) {
    auto node = node_of<DropoutBackward>(x, residual);
    node->counter = SavedVariable(counter, false);
    node->drop = drop;
    node->seed = seed;
    node->offset = offset;
    set_history(out, node);
  }
  return out;
}

Tensor dropout_add(const Tensor& x, const std::optional<Tensor>& residual_, double p, uint64_t seed,
                   uint64_t offset, const std::optional<Tensor>& counter_) {
  const Tensor residual = or_none(residual_), counter = or_none(counter_);
  check_tensors({&x, &residual, &counter});
  storage_code(x);
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == x.sizes() &&
                                            residual.scalar_type() == x.scalar_type()),
                    "residual ", residual.defined() ? residual.sizes() : x.sizes(),
                    " does not match x ", x.sizes(), " (sizes and dtype)");
  TORCH_CHECK_VALUE(!counter.defined() || (counter.scalar_type() == at::kLong && counter.numel() == 1),
                    "an offset tensor holds one int64");
  return dropout(x, residual, (int64_t)std::nearbyint(p * 65536), seed, offset, counter);
}

// ---------------------------------------------------------------- norm and rotation
xnn_heads heads_of(const Tensor& t) {
  return xnn_heads{t.data_ptr(), t.stride(0), t.stride(1), (int32_t)t.size(1)};
}

Tensor unit_stride(const Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); }

constexpr int64_t kMaxHeadDim = 128;

struct NormRotateBackward : Node {
  SavedVariable q, k, q_weight, k_weight, cos, sin, positions;
  double eps;
  bool interleaved;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable();
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const Tensor q = this->q.unpack(), k = this->k.unpack(), qw = q_weight.unpack(),
                 kw = k_weight.unpack(), c = cos.unpack(), s = sin.unpack(), pos = positions.unpack();
    const c10::DeviceGuard guard(q.device());
    const Tensor gq = grads[0].defined() ? grads[0].contiguous() : at::zeros(q.sizes(), q.options());
    const Tensor gk = grads[1].defined() ? grads[1].contiguous() : at::zeros(k.sizes(), k.options());
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    Tensor dqw, dkw, dc, ds, work;
    size_t need = 0;
    if (task_should_compute_output(2) || task_should_compute_output(3)) {
      dqw = at::empty(qw.sizes(), qw.options());
      dkw = at::empty(kw.sizes(), kw.options());
      check("xnn_head_norm_rotate_backward_work_size",
            api.xnn_head_norm_rotate_backward_work_size((int32_t)q.size(2), &need));
      work = bytes(q, need);
    }
    if (task_should_compute_output(4) || task_should_compute_output(5)) {
      dc = at::empty(c.sizes(), c.options());
      ds = at::empty(s.sizes(), s.options());
    }
    const xnn_heads qh = heads_of(q), kh = heads_of(k);
    XNN_CALL(xnn_head_norm_rotate_backward, storage_code(q), &qh, &kh, q.size(0), (int32_t)q.size(2),
             (int32_t)(2 * c.size(1)), data(qw), data(kw), c.const_data_ptr<float>(),
             s.const_data_ptr<float>(), c.size(0), (const int64_t*)data(pos), (float)eps, interleaved,
             data(gq), data(gk), data(dq), data(dk), data(dqw), data(dkw), (float*)data(dc),
             (float*)data(ds), data(work), need, stream_of(q));
    const Tensor all[] = {dq, dk, dqw, dkw, dc, ds};
    for (int i = 0; i < 6; ++i)
      if (task_should_compute_output(i)) out[i] = all[i];
    return out;
  }
  void release_variables() override {
    for (SavedVariable* v : {&q, &k, &q_weight, &k_weight, &cos, &sin, &positions}) v->reset_data();
  }
  std::string name() const override { return "XnnHeadNormRotateBackward"; }
};

std::tuple<Tensor, Tensor> head_norm_rotate(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos,
                                            Tensor sin, const std::optional<Tensor>& positions_, double eps,
                                            bool interleaved) {
  Tensor positions = or_none(positions_);
  check_tensors({&q, &k, &q_weight, &k_weight, &cos, &sin, &positions});
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                    "q and k must be (tokens, heads, head_dim) of the same tokens and head_dim, got ",
                    q.sizes(), " and ", k.sizes());
  const int64_t T = q.size(0), D = q.size(2);
  TORCH_CHECK_VALUE(D >= 1 && D <= kMaxHeadDim, "head_dim must be in [1, ", kMaxHeadDim, "], got ", D);
  TORCH_CHECK_VALUE(q.size(1) >= 1 && k.size(1) >= 1, "no heads");
  const int code = storage_code(q);
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
  const c10::DeviceGuard guard(q.device());
  if (!positions.defined()) {
    TORCH_CHECK_VALUE(cos.size(0) == T, "without positions the tables have a row a token: ", cos.size(0),
                      " rows, ", T, " tokens");
  } else {
    TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == T &&
                          at::isIntegralType(positions.scalar_type(), false),
                      "positions must be (", T, ",) integers");
    TORCH_CHECK_VALUE(!wanted({&cos, &sin}), "tables read by position have no gradient here (gather their "
                                             "rows and leave positions out)");
    positions = positions.to(at::kLong).contiguous();
  }
  q = unit_stride(q);
  k = unit_stride(k);
  q_weight = q_weight.contiguous();
  k_weight = k_weight.contiguous();
  cos = cos.contiguous();
  sin = sin.contiguous();
  Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
  const xnn_heads qh = heads_of(q), kh = heads_of(k);
  XNN_CALL(xnn_head_norm_rotate, code, &qh, &kh, T, (int32_t)D, (int32_t)(2 * cos.size(1)), data(q_weight),
           data(k_weight), cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), cos.size(0),
           (const int64_t*)data(positions), (float)eps, interleaved, data(q_out), data(k_out),
           stream_of(q));
  if (wanted({&q, &k, &q_weight, &k_weight, &cos, &sin})) {
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
    set_history(q_out, node);
    set_history(k_out, node);
  }
  return {q_out, k_out};
}

// ---------------------------------------------------------------- attention
struct Plan {
  int64_t n_tokens, max_atoms;
  Tensor tiles32, tiles128;
  xnn_attention_tiles tiles;
  Plan(int64_t n_tokens, int64_t max_atoms, const Tensor& tiles32, const Tensor& tiles128)
      : n_tokens(n_tokens), max_atoms(max_atoms), tiles32(tiles32), tiles128(tiles128) {
    tiles = xnn_attention_tiles{n_tokens,
                                max_atoms,
                                tiles32.size(0),
                                tiles128.size(0),
                                (const int32_t*)data(tiles32),
                                (const int32_t*)data(tiles128)};
  }
};

struct AttentionBackward : Node {
  SavedVariable q, k, v, mask, out, lse;
  std::shared_ptr<Plan> plan;
  double scale;
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable();
    variable_list result(3);
    if (!grads[0].defined()) return result;
    const Tensor q = this->q.unpack(), k = this->k.unpack(), v = this->v.unpack(), m = mask.unpack(),
                 o = out.unpack(shared_from_this()), l = lse.unpack();
    const c10::DeviceGuard guard(q.device());
    const Tensor g = grads[0].contiguous();
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                 dv = at::empty(v.sizes(), v.options());
    size_t need = 0;
    check("xnn_attention_backward_work_size",
          api.xnn_attention_backward_work_size(storage_code(q), q.size(0), (int32_t)q.size(1), (int32_t)k.size(1),
                                               (int32_t)q.size(2), &plan->tiles, &need));
    const Tensor work = bytes(q, need);
    const xnn_heads qh = heads_of(q), kh = heads_of(k), vh = heads_of(v);
    XNN_CALL(xnn_attention_backward, storage_code(q), &qh, &kh, &vh, q.size(0), (int32_t)q.size(2),
             &plan->tiles, (const uint8_t*)data(m), (float)scale, data(o), l.const_data_ptr<float>(), data(g),
             data(dq), data(dk), data(dv), data(work), need, stream_of(q));
    const Tensor all[] = {dq, dk, dv};
    for (int i = 0; i < 3; ++i)
      if (task_should_compute_output(i)) result[i] = all[i];
    return result;
  }
  void release_variables() override {
    for (SavedVariable* s : {&q, &k, &v, &mask, &out, &lse}) s->reset_data();
  }
  std::string name() const override { return "XnnAttentionBackward"; }
};

Tensor structure_attention(Tensor q, Tensor k, Tensor v, const std::shared_ptr<Plan>& plan,
                           const std::optional<Tensor>& mask_, const std::optional<double>& scale_) {
  Tensor mask = or_none(mask_);
  check_tensors({&q, &k, &v, &mask, &plan->tiles32});
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
                        q.size(2) == k.size(2),
                    "q must be (tokens, heads, head_dim), k and v (tokens, kv_heads, head_dim), got ",
                    q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  TORCH_CHECK_VALUE(D >= 1 && D <= kMaxHeadDim, "head_dim must be in [1, ", kMaxHeadDim, "], got ", D);
  TORCH_CHECK_VALUE(k.size(1) >= 1 && H >= 1 && H % k.size(1) == 0, H, " heads cannot share ", k.size(1),
                    " heads of keys and values");
  const int code = storage_code(q);
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k and v must have one dtype, got ", q.scalar_type(), ", ", k.scalar_type(), " and ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(plan->n_tokens == T, "the plan is of ", plan->n_tokens, " tokens, q holds ", T);
  const c10::DeviceGuard guard(q.device());
  if (mask.defined()) {
    TORCH_CHECK_VALUE(mask.dim() == 1 && mask.size(0) == T && mask.scalar_type() == at::kBool,
                      "mask must be (", T, ",) bool, got ", mask.sizes(), " ", mask.scalar_type());
    mask = mask.contiguous();
  }
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(scale > 0.0 && scale < std::numeric_limits<double>::infinity(),
                    "scale must be positive and finite, got ", scale);
  q = unit_stride(q);
  k = unit_stride(k);
  v = unit_stride(v);
  const bool train = wanted({&q, &k, &v});
  Tensor out = at::empty(q.sizes(), q.options()), lse, work;
  if (train) lse = at::empty({H, T}, q.options().dtype(at::kFloat));
  size_t need = 0;
  check("xnn_attention_work_size",
        api.xnn_attention_work_size(code, T, (int32_t)H, (int32_t)D, &plan->tiles, &need));
  if (need > 0) work = bytes(q, need);
  const xnn_heads qh = heads_of(q), kh = heads_of(k), vh = heads_of(v);
  XNN_CALL(xnn_attention, code, &qh, &kh, &vh, T, (int32_t)D, &plan->tiles, (const uint8_t*)data(mask),
           (float)scale, data(out), (float*)data(lse), data(work), need, stream_of(q));
  if (train) {
    auto node = node_of<AttentionBackward>(q, k, v);
    node->q = SavedVariable(q, false);
    node->k = SavedVariable(k, false);
    node->v = SavedVariable(v, false);
    node->mask = SavedVariable(mask, false);
    node->lse = SavedVariable(lse, false);
    node->plan = plan;
    node->scale = scale;
    set_history(out, node);
    node->out = SavedVariable(out, true);
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("load", &load);
  m.def("calls", &calls);
  m.def("embedding", &embedding);
  m.def("dropout_add", &dropout_add);
  m.def("head_norm_rotate", &head_norm_rotate);
  m.def("structure_attention", &structure_attention);
  py::class_<Plan, std::shared_ptr<Plan>>(m, "Plan")
      .def(py::init<int64_t, int64_t, const Tensor&, const Tensor&>());
}
