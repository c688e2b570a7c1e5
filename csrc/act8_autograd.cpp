// Autograd of linear_act8 in C++ (the host time of a backward through a Python function is most of a small layer's step).
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <string>
#include "act8.h"

namespace dmad {

using OptTensor = c10::optional<at::Tensor>;

void check_captured_backward(const std::string& op);

namespace {

struct LinearAct8 : torch::autograd::Function<LinearAct8> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const OptTensor& bias, int64_t act, bool keep) {
    auto [y, data, exponents] = act8_forward(x, w, bias, act, keep);
    const bool has_bias = bias.has_value() && bias->defined();
    ctx->save_for_backward({w, data, exponents});
    ctx->saved_data["act"] = act;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["bias"] = has_bias;
    ctx->saved_data["bias_type"] = (int64_t)(has_bias ? bias->scalar_type() : at::kFloat);
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    check_captured_backward("linear_act8");
    const auto s = ctx->get_saved_variables();
    const bool has_bias = ctx->saved_data["bias"].toBool();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
    torch::autograd::variable_list out(5);
    {
      at::NoGradGuard no_grad;
      auto [dx, dw, db] = act8_backward(g[0], s[0], s[1], s[2], ctx->saved_data["act"].toInt(), rows, ctx->needs_input_grad(0),
                                        ctx->needs_input_grad(1), has_bias && ctx->needs_input_grad(2),
                                        (at::ScalarType)ctx->saved_data["bias_type"].toInt());
      if (dx.defined()) dx = dx.view(shape);
      out[0] = dx;
      out[1] = dw;
      out[2] = db;
    }
    if (at::GradMode::is_enabled()) {  // a second derivative is an error and not a constant
      for (auto& t : out) {
        if (!t.defined()) continue;
        torch::autograd::variable_list from{t.set_requires_grad(true), s[0], g[0]};  // all that the gradient depends on
        auto error = std::make_shared<torch::autograd::DelayedError>("linear_act8 is differentiable once", (int64_t)from.size());
        t = (*error)(std::move(from))[0];
      }
    }
    return out;
  }
};

}  // namespace

at::Tensor linear_act8(const at::Tensor& x, const at::Tensor& w, OptTensor bias, int64_t act) {
  act8_check(x, w, bias, act);
  const bool db = bias.has_value() && bias->defined() && bias->requires_grad();
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || w.requires_grad() || db))
    return std::get<0>(act8_forward(x, w, bias, act, false));
  // the input is kept for the weight's gradient, and for the activation's derivative
  return LinearAct8::apply(x, w, bias, act, w.requires_grad() || (act != kActNone && x.requires_grad()));
}

}  // namespace dmad
