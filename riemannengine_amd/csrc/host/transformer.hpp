// What the autograd functions of the transformer operators share: streams,
// buffers, types and views of their tensors.
#pragma once

#include <ATen/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "riemann.hpp"

namespace riemann {

using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

inline hipStream_t stream_of(const at::Device &dev) {
  return c10::hip::getCurrentHIPStream(dev.index()).stream();
}

inline at::Tensor byte_buffer(size_t bytes, const at::Device &dev) {
  return torch::empty({static_cast<int64_t>(bytes)},
                      torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

inline int32_t hip_dtype(const at::Tensor &t, const char *what) {
  if (t.scalar_type() == torch::kBFloat16)
    return RHIP_BF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat, what, " must be fp32 or bf16, got ",
              t.scalar_type());
  return RHIP_F32;
}

// Optional tensors travel through autograd as empty tensors.
inline bool present(const at::Tensor &t) { return t.defined() && t.numel() > 0; }
inline at::Tensor or_empty(const at::Tensor &t, const at::Tensor &like) {
  return t.defined() ? t : torch::empty({0}, like.options());
}
inline const float *fptr(const at::Tensor &t) { return present(t) ? t.data_ptr<float>() : nullptr; }
inline float *fptr_mut(at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
inline void *vptr_mut(at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The kernels take any strides but a strided last axis.
inline at::Tensor dense_last(const at::Tensor &t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

inline at::Tensor int_vector(const at::Tensor &t, const at::Device &dev, const char *what) {
  TORCH_CHECK(t.device() == dev, what, " must be on the queries' device");
  TORCH_CHECK(t.dim() == 1 && (t.scalar_type() == torch::kInt || t.scalar_type() == torch::kLong),
              what, " must be a vector of int32 or int64");
  return t.to(torch::kInt).contiguous();
}

// Whether a call goes through its autograd function: an input is recorded, or
// carries a forward-mode tangent (which the function refuses; without it the
// result would lose the tangent).
inline bool through_autograd(std::initializer_list<at::Tensor> ts) {
  for (const auto &t : ts)
    if (t.defined() && ((torch::GradMode::is_enabled() && t.requires_grad()) ||
                        t._fw_grad(0).defined()))
      return true;
  return false;
}

// The gradients come from kernels that autograd does not see: a second
// derivative would silently lack them.
inline void first_derivative_only(const char *what) {
  TORCH_CHECK(!torch::GradMode::is_enabled(), what,
              " has no second derivatives (backward with create_graph)");
}
// The same where a backward with create_graph may go through: its gradients, of
// what `on` holds, refuse to be differentiated themselves.
inline tensor_list not_twice(tensor_list grads, const tensor_list &on, const char *what) {
  if (!torch::GradMode::is_enabled())
    return grads;
  const size_t n = grads.size();
  grads.insert(grads.end(), on.begin(), on.end());
  auto refusal = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " has no second derivatives", static_cast<int64_t>(grads.size()));
  grads = (*refusal)(std::move(grads));
  grads.resize(n);
  return grads;
}

} // namespace riemann
