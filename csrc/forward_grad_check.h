// Forward-mode derivatives: the operators have reverse-mode gradients only.
#pragma once

#include <ATen/ATen.h>

#include <initializer_list>

namespace st {

// A tensor can carry a tangent without requiring a gradient; below autograd that tangent would be
// dropped and the derivative come out as zero, so such a call is refused.
inline void refuse_forward_grad(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                              ": forward-mode derivatives are not implemented (an input has a tangent)");
}
inline void refuse_forward_grad(at::TensorList inputs, const char* name) {
  for (const auto& t : inputs) refuse_forward_grad(t, name);
}
inline void refuse_forward_grad(std::initializer_list<const at::Tensor*> inputs, const char* name) {
  for (const at::Tensor* t : inputs)
    if (t) refuse_forward_grad(*t, name);
}

}  // namespace st
