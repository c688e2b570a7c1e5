// Rows of bf16, fp16 or fp32 numbers in units of 16 elements, as the quantisers read them.
#pragma once
#include <cstdint>
#include <type_traits>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "sm100.cuh"

namespace dmad {

// 32-byte accesses (whole sectors; 32-byte aligned addresses).
__device__ __forceinline__ void ld256(const void* p, uint32_t* w) {
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void st256(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 16 bytes that are read once: past the L1.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

constexpr uint32_t kInfBits = 0x7f800000u;  // non-negative fp32 numbers from here on are infinity and NaN

template <typename T>
struct Unit {  // 16 elements
  uint32_t w[4 * sizeof(T)];
};

template <typename T, bool ALIGNED>
__device__ __forceinline__ Unit<T> load_unit(const T* __restrict__ row, int c0, int K) {
  Unit<T> u;
  if constexpr (ALIGNED) {  // K is a multiple of 16: a unit is inside the row or past it
    if (c0 < K) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ld256(row + c0 + i * 32 / (int)sizeof(T), u.w + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 4 * (int)sizeof(T); ++i) u.w[i] = 0u;
    }
  } else if constexpr (sizeof(T) == 4) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(row);
#pragma unroll
    for (int i = 0; i < 16; ++i) u.w[i] = c0 + i < K ? __ldg(p + c0 + i) : 0u;
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = c0 + 2 * i < K ? __ldg(p + c0 + 2 * i) : 0u;
      const uint32_t hi = c0 + 2 * i + 1 < K ? __ldg(p + c0 + 2 * i + 1) : 0u;
      u.w[i] = lo | (hi << 16);
    }
  }
  return u;
}

// max |x| of a unit as the bits of an fp32 number.  Non-negative numbers order as their bits do, with infinity
// and NaN above all finite ones (16-bit maxima carry a NaN on).
template <typename T>
__device__ __forceinline__ uint32_t absmax_bits(const Unit<T>& u) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, u.w[i] & 0x7fffffffu);
    return m;
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.w[i])));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&m) & 0x7fff7fffu;
    return max(w & 0xffffu, w >> 16) << 16;
  } else {
    __half2 m = __habs2(*reinterpret_cast<const __half2*>(&u.w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&u.w[i])));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&m) & 0x7fff7fffu;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(w & 0xffffu, w >> 16))));
  }
}

// Elements 2i and 2i + 1 of a unit as two packed floats.
template <typename T>
__device__ __forceinline__ uint64_t unit_pair(const Unit<T>& u, int i) {
  if constexpr (sizeof(T) == 4) {
    return f2(__uint_as_float(u.w[2 * i]), __uint_as_float(u.w[2 * i + 1]));
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return f2(__uint_as_float(u.w[i] << 16), __uint_as_float(u.w[i] & 0xffff0000u));
  } else {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&u.w[i]));
    return f2(h.x, h.y);
  }
}

}  // namespace dmad
