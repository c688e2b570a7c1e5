// Argument checks that end in a Python ValueError, like those of the Python wrappers.  (The latency of a call on
// one token is that of its host code, so the CUDA paths check their arguments here and not in Python as well.)
#pragma once
#include <torch/extension.h>
#include <array>
#include <atomic>
#include <cuda_runtime.h>
#include <string>

namespace dmad {

#define DMAD_VALUE_CHECK(cond, msg)                              \
  do {                                                           \
    if (!(cond)) throw pybind11::value_error(std::string(msg));  \
  } while (0)

inline const char* dtype_name(at::ScalarType t) {
  return t == at::kBFloat16 ? "bf16" : t == at::kHalf ? "fp16" : t == at::kFloat ? "fp32" : "another type";
}

inline bool is_float_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

// Shape as text, "(4, 64)".
inline std::string shape_text(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

// Multiprocessors of a device, asked for once.
inline int sm_count(int device) {
  static std::array<std::atomic<int>, 64> known{};
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    n = 148;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace dmad
