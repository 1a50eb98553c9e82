// Checks of autograd operators under graph capture.
#pragma once
#include <torch/extension.h>

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/variable.h>

namespace ddb {

inline bool capturing() { return at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None; }

// A backward pass that is captured while an eager graph of the same leaf is alive ends the
// process inside autograd: the leaf's accumulation node belongs to the default stream.
inline void refuse_eager_leaf(const torch::Tensor& t) {
  if (!t.requires_grad() || !t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto s = node->stream();
  TORCH_CHECK(!s || c10::cuda::CUDAStream(*s).stream() != nullptr,
              "an autograd graph made on the default stream still uses this leaf: drop it before capturing a backward "
              "pass, or warm up on another stream");
}

}  // namespace ddb
