// Host side of the 8-bit operators: a stored matrix, its checks, and the launchers.
#pragma once
#include "checks.h"
#include "int8.cuh"

namespace dmad {

// Threads of a row (whole warps, as even a share of the row's units each as there is) and rows of a block of up to 256.
inline dim3 row_block(int64_t units) {
  const int64_t passes = (units + 255) / 256;
  const unsigned tx = (unsigned)std::max<int64_t>(32, ((units + passes - 1) / passes + 31) / 32 * 32);
  return dim3(tx, 256 / tx);
}

struct Int8Matrix {  // storage as int8.cuh describes it
  int8_t* data;
  float* row_scale;    // one scale a row
  uint8_t* exponents;  // blocks of 32
  int64_t rows, cols;

  int64_t row_bytes() const { return int8_row_bytes(cols); }
  int64_t blocks() const { return (cols + kInt8Block - 1) / kInt8Block; }
};

// The matrix behind data / scale [rows, cols] on `device`; a ValueError where they do not fit.
Int8Matrix int8_matrix(const at::Tensor& data, const at::Tensor& scale, int64_t rows, int64_t cols, bool blocks,
                       const at::Device& device, const char* name);

// x [..., K] as a matrix [R, K] with contiguous columns.
at::Tensor int8_rows(const at::Tensor& x, const char* name);

// x [rows, cols] (contiguous columns) -> q, whose memory the caller provides (row_scale or exponents).
void int8_quantize_launch(const at::Tensor& x, const Int8Matrix& q, cudaStream_t stream);


// The values of q -> out [rows, cols] (bf16, fp16 or fp32, contiguous columns, rows at any distance).
void int8_dequantize_launch(const Int8Matrix& q, const at::Tensor& out, cudaStream_t stream);

}  // namespace dmad
