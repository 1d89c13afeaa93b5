// Whether an operator's autograd node is needed: what the operators' Autograd kernels ask first.
#pragma once
#include <torch/csrc/autograd/functions/utils.h>

#include "torch_common.h"

namespace mi355_torch {

inline bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }

// Operators have backward formulas only.  A tangent (torch.autograd.forward_ad, torch.func.jvp) is no matter of requires_grad, and
// below Autograd it would be lost without a word: refused here, in front of any launch.
template <typename... Ts>
bool differentiated(const char* name, const Ts&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), "mi355_moe::", name, " has no forward-mode derivative");
  return torch::autograd::compute_requires_grad(inputs...);
}

}  // namespace mi355_torch
