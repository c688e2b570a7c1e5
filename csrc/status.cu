// Device status word shared by every kernel with bounded waits.  Kernels write
// the first failure code (see DeviceStatus in sm100.cuh) instead of trapping;
// the host polls it with device_status() after a step and raises.
#include <cuda_runtime.h>
#include <torch/extension.h>
#include <c10/cuda/CUDAException.h>
#include <mutex>
#include <vector>

namespace dmad {

int* device_status_ptr(int device) {
  static std::mutex mu;
  static std::vector<int*> ptrs;
  std::lock_guard<std::mutex> lock(mu);
  if ((int)ptrs.size() <= device) ptrs.resize(device + 1, nullptr);
  if (ptrs[device] == nullptr) {
    // The first kernel of a process may be one that a graph captures: the word is made outside of the capture, on a
    // stream of its own.
    int prev;
    C10_CUDA_CHECK(cudaGetDevice(&prev));
    C10_CUDA_CHECK(cudaSetDevice(device));
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    int* word = nullptr;
    cudaStream_t stream = nullptr;
    cudaError_t err = cudaMalloc(&word, sizeof(int));
    if (err == cudaSuccess) err = cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
    if (err == cudaSuccess) err = cudaMemsetAsync(word, 0, sizeof(int), stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
    if (stream != nullptr) cudaStreamDestroy(stream);
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    C10_CUDA_CHECK(cudaSetDevice(prev));
    C10_CUDA_CHECK(err);
    ptrs[device] = word;
  }
  return ptrs[device];
}

// Returns the status code of `device` (synchronising with it) and optionally clears it.
int64_t device_status(int64_t device, bool reset) {
  int* p = device_status_ptr((int)device);
  int prev;
  C10_CUDA_CHECK(cudaGetDevice(&prev));
  C10_CUDA_CHECK(cudaSetDevice((int)device));
  int v = 0;
  C10_CUDA_CHECK(cudaMemcpy(&v, p, sizeof(int), cudaMemcpyDeviceToHost));
  if (reset) C10_CUDA_CHECK(cudaMemset(p, 0, sizeof(int)));
  C10_CUDA_CHECK(cudaSetDevice(prev));
  return v;
}

}  // namespace dmad
