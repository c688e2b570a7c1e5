// Integer codes of 8 bits: the storage layout that the quantiser, the products and the trained linear layer share, and
// the conversions.
//
// A matrix [R, K] is stored as
//   data    [R, ceil(K / 32) * 32] signed bytes, -127 .. 127; columns past K are zero.
//   scale   one scale a row: fp32 [R], s = max|x| / 127, from 2^-126 to 0x1.020406p121 (whose
//           127-fold is finite), 1 for a row of zeros, NaN for a row with an
//           infinity or a NaN (whose codes are 0);
//           blocks of 32 columns: bytes [R, ceil(K / 32)], the biased exponent of s = 2^(floor(log2 max|x|) - 6), at least
//           0 (2^-127); 255 (NaN) for a block with an infinity or a NaN, 0 for one of zeros.
// A code is x / s rounded to the nearest whole number, halves to the even one; blocks clip +-128 to +-127.  Every code is
// decided exactly, so that it depends on the numbers alone.
#pragma once
#include <cstdint>
#include "row_units.cuh"

namespace dmad {

constexpr int kInt8Block = 32;
constexpr float kInt8MinScale = 0x1p-126f, kInt8MaxScale = 0x1.020406p121f;
__host__ __device__ constexpr int64_t int8_row_bytes(int64_t K) { return (K + 31) / 32 * 32; }

// 1.5 * 2^23: adding it rounds |v| < 2^22 to a whole number (halves to the even one), which is then in the low bits.
constexpr float kRoundMagic = 12582912.f;

// Four whole numbers v + kRoundMagic -> their low bytes.
__device__ __forceinline__ uint32_t pack_bytes(uint64_t ab, uint64_t cd) {
  const uint32_t a = (uint32_t)ab, b = (uint32_t)(ab >> 32), c = (uint32_t)cd, d = (uint32_t)(cd >> 32);
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Scale of a row with the maximum amax (bits of an fp32 number); inv: 1 / s, rounded, and 0 for a row that is not finite.
__device__ __forceinline__ float int8_row_scale(uint32_t amax, float& inv) {
  if (amax >= kInfBits) {
    inv = 0.f;
    return __uint_as_float(0x7fffffffu);
  }
  const float s = amax == 0u ? 1.f : fminf(fmaxf(__fdiv_rn(__uint_as_float(amax), 127.f), kInt8MinScale), kInt8MaxScale);
  inv = __frcp_rn(s);
  return s;
}

// Four signed bytes -> two pairs of floats: the byte plus 128 in the low bits of 2^23, less 2^23 + 128.
__device__ __forceinline__ void bytes_to_float(uint32_t w, uint64_t& lo, uint64_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const uint64_t c = f2(-8388736.f, -8388736.f);
  const uint32_t m = 0x4b000000u;
  lo = f2_add(f2(__uint_as_float(__byte_perm(u, m, 0x7440)), __uint_as_float(__byte_perm(u, m, 0x7441))), c);
  hi = f2_add(f2(__uint_as_float(__byte_perm(u, m, 0x7442)), __uint_as_float(__byte_perm(u, m, 0x7443))), c);
}

// 2^(code - 127) of a block's scale byte (255: NaN).
__device__ __forceinline__ float int8_block_scale(uint32_t code) {
  return __uint_as_float(code == 0xffu ? 0x7fffffffu : code == 0u ? 0x00400000u : code << 23);
}
// Scale byte of a block with the maximum amax (bits of an fp32 number).
__device__ __forceinline__ uint32_t int8_block_code(uint32_t amax) {
  return amax >= kInfBits ? 0xffu : (uint32_t)max((int)(amax >> 23) - 6, 0);
}

__device__ __forceinline__ float clamp127(float v) {  // the sign of v, the smaller size of v and 127
  float r;
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(127.f));
  return r;
}

// Codes of 16 elements of a block with the scale byte `code`: x 2^(127 - code) is exact (a power of two of at most 2^127,
// |x| below 2^7 of its inverse).
template <typename T>
__device__ __forceinline__ void int8_encode_block(const Unit<T>& u, uint32_t code, uint32_t (&out)[4]) {
  if (code == 0xffu) {
    out[0] = out[1] = out[2] = out[3] = 0u;
    return;
  }
  const float m = __uint_as_float((254u - code) << 23);
  const uint64_t m2 = f2(m, m), c = f2(kRoundMagic, kRoundMagic);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint64_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 t = f2_split(f2_mul(unit_pair(u, 2 * q + h), m2));
      v[h] = f2_add(f2(clamp127(t.x), clamp127(t.y)), c);
    }
    out[q] = pack_bytes(v[0], v[1]);
  }
}

// x / s to the nearest whole number, halves to the even one, given n next to it: x - n s is exact (a multiple of the last
// place of x or s, and no larger than s).
__device__ __forceinline__ float exact_code(float x, float s, float n) {
  const float r = fmaf(-n, s, x), d = 2.f * fabsf(r);
  if (d > s || (d == s && ((int)n & 1))) n += copysignf(1.f, r);
  return n;
}

// Codes of 16 elements of a row with the scale s and inv = 1 / s, rounded.  x inv is off by at most 2^-16, so only
// quotients closer than that to a half are decided by their remainders.
template <typename T>
__device__ __forceinline__ void int8_encode_row(const Unit<T>& u, float s, float inv, uint32_t (&out)[4]) {
  const uint64_t i2 = f2(inv, inv), c = f2(kRoundMagic, kRoundMagic);
  float far = 0.f;  // the largest distance from a whole number
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint64_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint64_t t = f2_mul(unit_pair(u, 2 * q + h), i2);
      v[h] = f2_add(t, c);
      const float2 d = f2_split(f2_sub(t, f2_sub(v[h], c)));
      far = fmax3(far, fabsf(d.x), fabsf(d.y));
    }
    out[q] = pack_bytes(v[0], v[1]);
  }
  if (far > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint64_t v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t x = unit_pair(u, 2 * q + h);
        const float2 n = f2_split(f2_sub(f2_add(f2_mul(x, i2), c), c)), xs = f2_split(x);
        v[h] = f2_add(f2(exact_code(xs.x, s, n.x), exact_code(xs.y, s, n.y)), c);
      }
      out[q] = pack_bytes(v[0], v[1]);
    }
  }
}

}  // namespace dmad
