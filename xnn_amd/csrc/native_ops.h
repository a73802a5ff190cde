// What the registered operators share (host code): the library's entry points with the counts of their calls,
// checks of tensors, and the pieces of autograd nodes. A source names its entry points (XNN_ENTRIES) and its
// family of operators (XNN_FAMILY) before it includes this, and is an extension module of its own.
#pragma once
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
                                "the xnn_amd " XNN_FAMILY " operators have no forward-mode derivative");
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

typedef std::optional<Tensor> MaybeTensor;

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// ---------------------------------------------------------------- registration
#define XNN_IMPL_KERNEL(schema, f) m.impl(#schema, &f##_kernel);
#define XNN_IMPL_SHAPE(schema, f) m.impl(#schema, &f##_shape);
#define XNN_IMPL_REFUSE(schema, f) \
  m.impl(#schema, torch::CppFunction::makeFromBoxedFunction<&refuse_batches>());

// No rule for a batch of calls. (A batch of cotangents is a loop over the backward operators.)
void refuse_batches(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().name(), " has no batching rule (vmap)");
}

}  // namespace
