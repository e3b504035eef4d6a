// Forward-mode derivatives: the operators have reverse-mode gradients only.
#pragma once

#include <torch/csrc/autograd/forward_grad.h>
#include <ATen/ATen.h>

#include <initializer_list>

namespace st {

// A tensor can carry a tangent without requiring a gradient; below autograd that tangent would be
// dropped and the derivative come out as zero, so such a call is refused.
inline void refuse_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                              ": forward-mode derivatives are not implemented (an input has a tangent)");
}
// Tangents exist only while a dual level is open; else no tensor is looked at.
inline bool in_forward_mode() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
inline void refuse_forward_grad(std::initializer_list<const at::Tensor*> inputs, const char* name) {
  if (!in_forward_mode()) return;
  for (const at::Tensor* t : inputs)
    if (t) refuse_tangent(*t, name);
}
inline void refuse_forward_grad(std::initializer_list<at::TensorList> inputs, const char* name) {
  if (!in_forward_mode()) return;
  for (const at::TensorList l : inputs)
    for (const auto& t : l) refuse_tangent(t, name);
}

}  // namespace st
