// The linear layer that keeps its input in 8 bits: the parts that its autograd node calls.
#pragma once
#include <torch/extension.h>
#include <tuple>

namespace dmad {

enum Act8 : int { kActNone = 0, kActGelu = 1, kActSwiglu = 2 };

void act8_check(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& bias, int64_t act);
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_forward(const at::Tensor& x, const at::Tensor& w,
                                                            const c10::optional<at::Tensor>& bias, int64_t act, bool keep);
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_backward(const at::Tensor& g, const at::Tensor& w, const at::Tensor& data,
                                                             const at::Tensor& exponents, int64_t act, int64_t R,
                                                             bool want_x, bool want_w, bool want_b, at::ScalarType bias_type);

}  // namespace dmad
