// What the extension module's sources share (torch_ops.cpp, mixer_ops.cpp): streams,
// status checks, pointers and casts over the C ABI.
#pragma once
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "../../include/lizard_hip.h"

// The recurrent mixers' operators (mixer_ops.cpp)
void bind_mixers(pybind11::module_& m);

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline void check(int rc, const char* what) {
  if (rc != 0)
    throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(rc) +
                             "): " + lz_last_error());
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() && t.numel() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

inline Tensor as(const Tensor& t, at::ScalarType dtype) {
  return (t.scalar_type() == dtype ? t : t.to(dtype)).contiguous();
}
inline Tensor bf16(const Tensor& t) { return as(t, at::kBFloat16); }
inline Tensor f32(const Tensor& t) { return as(t, at::kFloat); }

inline Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

inline int i32(int64_t x) { return static_cast<int>(x); }

inline bool any_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

}  // namespace
