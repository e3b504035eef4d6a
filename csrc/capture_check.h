// A training call under graph capture while an earlier autograd graph of the same leaves is alive.
#pragma once

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/variable.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <initializer_list>

namespace st {

inline bool is_capturing(const c10::hip::HIPStream& stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(stream.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}

// A leaf's gradient is accumulated on the stream on which its accumulator was made, and an earlier
// graph that is still held keeps that accumulator.  A captured backward pass would make that other stream
// wait on the capture, which breaks the capture and ends the process from the engine's thread: such a
// call is refused before it records anything.  The stream is the current one of the tensor's device, which
// need not be the current device.
inline void check_capture(std::initializer_list<const at::Tensor*> inputs, const char* name) {
  for (const at::Tensor* t : inputs) {
    if (!t || !t->defined() || !t->requires_grad() || t->grad_fn() || !t->is_cuda()) continue;
    const auto current = c10::hip::getCurrentHIPStream(t->device().index());
    if (!is_capturing(current)) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream.has_value() || stream->id() == current.unwrap().id(), name,
                ": captured while an earlier autograd graph of an input is alive, whose gradients belong to another "
                "stream; delete that graph's outputs before the capture");
  }
}

}  // namespace st
