// Host side of the 4-bit operators: a stored matrix, its checks, and the launchers.
#pragma once
#include "checks.h"
#include "fp4.cuh"

namespace dmad {

struct Fp4Matrix {  // storage as fp4.cuh describes it
  uint8_t* data;
  uint8_t* scales;
  float* row_scale;  // nvfp4
  int64_t rows, cols;
  bool nv;

  int64_t row_bytes() const { return (cols + 31) / 32 * 16; }
  int64_t ktiles() const {
    const int64_t b = fp4_block(nv);
    return ((cols + b - 1) / b + kFp4TileBlocks - 1) / kFp4TileBlocks;
  }
  int64_t row_tiles() const { return (rows + kFp4TileRows - 1) / kFp4TileRows; }
  int64_t data_bytes() const { return rows * row_bytes(); }
  int64_t scale_bytes() const { return row_tiles() * ktiles() * kFp4TileBytes; }
};

// The matrix behind data / scales / row_scale [rows, cols] on `device`; a ValueError where they do not fit.
Fp4Matrix fp4_matrix(const at::Tensor& data, const at::Tensor& scales, const c10::optional<at::Tensor>& row_scale,
                     int64_t rows, int64_t cols, bool nv, const at::Device& device, const char* name);

// x [rows, cols] (contiguous columns) -> q, whose memory the caller provides.
void fp4_quantize_launch(const at::Tensor& x, const Fp4Matrix& q, cudaStream_t stream);

}  // namespace dmad
