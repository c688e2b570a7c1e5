// Autograd of qk_head_norm_rope in C++: a backward through a Python function costs the host some 50 us more, which for
// few rows is most of the step.
#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <stdexcept>
#include <string>

namespace dmad {

using OptTensor = c10::optional<at::Tensor>;

std::tuple<at::Tensor, at::Tensor> head_norm_rope_fwd(const at::Tensor& q, const at::Tensor& k, OptTensor wq, OptTensor wk,
                                                      OptTensor cosT, OptTensor sinT, OptTensor positions, double eps,
                                                      bool interleaved);
void head_norm_rope_bwd(const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k, OptTensor wq,
                        OptTensor wk, OptTensor cosT, OptTensor sinT, OptTensor positions, at::Tensor& dq, at::Tensor& dk,
                        OptTensor dwq, OptTensor dwk, double eps, bool interleaved);

// In a backward that a CUDA graph captures: an error where a leaf's gradient belongs to the default stream.  While an eager
// graph of the same leaves lives, they keep the accumulators that it made, and with them the stream on which it made
// them; the engine then makes that stream wait for the captured one.  Another stream joins the capture by that and is
// joined again at the end; the default stream cannot: no capture survives it, and the process may not either.
void check_captured_backward(const std::string& op) {
  const auto current = c10::cuda::getCurrentCUDAStream();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (current.stream() == nullptr || cudaStreamIsCapturing(current.stream(), &status) != cudaSuccess ||
      status != cudaStreamCaptureStatusActive)
    return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  for (const auto& edge : node->next_edges()) {
    auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get());
    if (leaf == nullptr) continue;
    const auto stream = leaf->stream();
    if (stream.has_value() && c10::cuda::CUDAStream(*stream).stream() == nullptr)
      throw std::runtime_error(op + ": this backward is being captured while a graph of the same leaves, recorded on the "
                                    "default stream, is alive; release that graph first, or record it on another stream");
  }
}

namespace {

OptTensor given(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

struct HeadNormRope : torch::autograd::Function<HeadNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const at::Tensor& k, const OptTensor& wq, const OptTensor& wk,
                                                const OptTensor& cosT, const OptTensor& sinT, const OptTensor& positions,
                                                double eps, bool interleaved) {
    auto [qo, ko] = head_norm_rope_fwd(q, k, wq, wk, cosT, sinT, positions, eps, interleaved);
    auto or_none = [](const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); };
    ctx->save_for_backward({q, k, or_none(wq), or_none(wk), or_none(cosT), or_none(sinT), or_none(positions)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {qo, ko};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    check_captured_backward("qk_head_norm_rope");
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(9);
    {
      at::NoGradGuard no_grad;
      const auto plain = [](const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); };
      out[0] = plain(s[0]);
      out[1] = plain(s[1]);
      for (int i = 2; i < 4; ++i)
        if (s[i].defined() && s[i].requires_grad()) out[i] = plain(s[i]);
      head_norm_rope_bwd(g[0], g[1], s[0], s[1], given(s[2]), given(s[3]), given(s[4]), given(s[5]), given(s[6]), out[0],
                         out[1], given(out[2]), given(out[3]), ctx->saved_data["eps"].toDouble(),
                         ctx->saved_data["interleaved"].toBool());
    }
    if (at::GradMode::is_enabled()) {  // a second derivative is an error and not a constant
      for (auto& t : out) {
        if (!t.defined()) continue;
        torch::autograd::variable_list from{t.set_requires_grad(true)};  // all that the gradient depends on
        for (int i = 0; i < 4; ++i)
          if (s[i].defined()) from.push_back(s[i]);
        from.insert(from.end(), g.begin(), g.end());
        auto error = std::make_shared<torch::autograd::DelayedError>("qk_head_norm_rope is differentiable once",
                                                                     (int64_t)from.size());
        t = (*error)(std::move(from))[0];
      }
    }
    return out;
  }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> head_norm_rope(const at::Tensor& q, const at::Tensor& k, OptTensor wq, OptTensor wk,
                                                  OptTensor cosT, OptTensor sinT, OptTensor positions, double eps,
                                                  bool interleaved) {
  auto out = HeadNormRope::apply(q, k, wq, wk, cosT, sinT, positions, eps, interleaved);
  return {out[0], out[1]};
}

}  // namespace dmad
