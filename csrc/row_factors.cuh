// acc ra rb + bias for the factors of a row and of a column, without an overflow or a lost digit where the result has
// none.  An accumulator is 0 or of a size from 2^-20 (nvfp4: two codes and two scales) to 2^47 (K <= 2^24 products of at
// most (6 * 448)^2; 8-bit integers: 1 to 2^31), so acc ra is an ordinary number for ra from 2^-80 to 2^80 and the last step
// rounds once.  For rows further out (elements above 1e27, or all below 1e-20) rb comes first, on acc c with c = 2^+-64,
// and ra / c last: acc c rb is larger than fp32 only if the result is, and small enough to lose digits only if the result is
// below 2^-140.
#pragma once
#include <cuda_runtime.h>

namespace dmad {

__device__ __forceinline__ bool far_out(float ra) { return !(ra >= 0x1p-80f && ra <= 0x1p80f); }
__device__ __forceinline__ float apply_factors(float acc, float ra, float rb, float bias) {
  return fmaf(acc * ra, rb, bias);
}
__device__ __forceinline__ float apply_factors_far(float acc, float ra, float rb, float bias) {
  const bool big = ra > 1.f;
  return fmaf(acc * (big ? 0x1p64f : 0x1p-64f) * rb, ra * (big ? 0x1p-64f : 0x1p64f), bias);
}

}  // namespace dmad
