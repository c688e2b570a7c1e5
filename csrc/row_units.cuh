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

// Rows that start anywhere (16 columns from c0, a multiple of 16, on): the 32-byte pieces around the unit, which are inside of
// the row except at its ends, moved into place by the row's offset (the same for a warp).  Where a piece reaches past the row
// its elements are read one by one.
template <typename T>
__device__ __forceinline__ void load_piece(const T* __restrict__ row, int c, int K, uint32_t* w) {  // 32 bytes from column c on
  constexpr int kElements = 32 / (int)sizeof(T);
  if (c >= 0 && c + kElements <= K) {
    ld256(row + c, w);
  } else if constexpr (sizeof(T) == 4) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = c + i >= 0 && c + i < K ? __ldg(p + c + i) : 0u;
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = c + 2 * i;
      const uint32_t lo = k >= 0 && k < K ? __ldg(p + k) : 0u, hi = k + 1 >= 0 && k + 1 < K ? __ldg(p + k + 1) : 0u;
      w[i] = lo | (hi << 16);
    }
  }
}

template <typename T>
__device__ __forceinline__ Unit<T> load_unit_anywhere(const T* __restrict__ row, int c0, int K) {
  constexpr int kPieces = (int)sizeof(T) / 2 + 1, kElements = 32 / (int)sizeof(T), kWords = 4 * (int)sizeof(T);
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 31);
  const int before = (int)(off / sizeof(T));
  uint32_t w[8 * kPieces + 1];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) load_piece(row, c0 - before + i * kElements, K, w + 8 * i);
  w[8 * kPieces] = 0u;
  Unit<T> u;
  const uint32_t odd = sizeof(T) == 2 ? (off & 2) * 8 : 0u;  // bits
  auto move = [&](auto words) {
    constexpr int n = decltype(words)::value;
#pragma unroll
    for (int i = 0; i < kWords; ++i) u.w[i] = __funnelshift_r(w[i + n], w[i + n + 1], odd);
  };
  switch (off >> 2) {
    case 0: move(std::integral_constant<int, 0>{}); break;
    case 1: move(std::integral_constant<int, 1>{}); break;
    case 2: move(std::integral_constant<int, 2>{}); break;
    case 3: move(std::integral_constant<int, 3>{}); break;
    case 4: move(std::integral_constant<int, 4>{}); break;
    case 5: move(std::integral_constant<int, 5>{}); break;
    case 6: move(std::integral_constant<int, 6>{}); break;
    default: move(std::integral_constant<int, 7>{}); break;
  }
  return u;
}

// The other way: a warp's 32 units of 16-bit results (16 columns each, of the lane from c0 on) to a row that starts anywhere.
// Each lane writes the aligned piece that begins in the lane before; the elements at the warp's ends, and at the row's, go one
// by one.  All lanes of the warp take part.
__device__ __forceinline__ void store_unit_anywhere(uint16_t* row, int c0, int K, const uint32_t (&r)[8]) {
  const int lane = lane_id();
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 31);
  const int before = (int)(off >> 1);
  uint32_t w[17];  // the lane before's words, then this lane's
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = __shfl_up_sync(0xffffffffu, r[i], 1);
    w[8 + i] = r[i];
  }
  w[16] = 0u;
  uint32_t o[8];
  const uint32_t odd = off & 2 ? 16u : 0u;  // o = 16 elements from element 16 - before of w on
  auto move = [&](auto words) {
    constexpr int n = 8 - decltype(words)::value;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = odd ? __funnelshift_r(w[i + n - 1], w[i + n], 16) : w[i + n];
  };
  switch (off >> 2) {
    case 0: move(std::integral_constant<int, 0>{}); break;
    case 1: move(std::integral_constant<int, 1>{}); break;
    case 2: move(std::integral_constant<int, 2>{}); break;
    case 3: move(std::integral_constant<int, 3>{}); break;
    case 4: move(std::integral_constant<int, 4>{}); break;
    case 5: move(std::integral_constant<int, 5>{}); break;
    case 6: move(std::integral_constant<int, 6>{}); break;
    default: move(std::integral_constant<int, 7>{}); break;
  }
  const int c = c0 - before;  // first column of the piece; lane 0 has the columns from c0 on only
  if ((lane > 0 || before == 0) && c + 16 <= K) {
    st256(row + c, o);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = c + i;
      if ((lane > 0 || k >= c0) && k < K) row[k] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
    }
  }
  if (lane == 31) {  // the columns that the next warp's first lane leaves to this one
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      const int k = c0 + i;
      if (i >= 16 - before && k < K) row[k] = (uint16_t)(r[i >> 1] >> (16 * (i & 1)));
    }
  }
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
