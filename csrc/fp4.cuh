// Block-scaled 4-bit floating point: the storage layout shared by the quantiser and the GEMM, and the
// sm_100a instructions that convert and multiply e2m1 numbers.
//
// A matrix [R, K] is stored as
//   data       [R, ceil(K / 32) * 16] bytes: two e2m1 codes a byte, the even column in the low four bits;
//              columns past K are zero.  Rows are multiples of 16 bytes, as TMA wants them.
//   scales     one byte a block of kBlock columns (mxfp4: 32, ue8m0; nvfp4: 16, e4m3), in tiles of
//              128 rows x 4 blocks of 512 bytes: byte (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4.  This is
//              the order in which tcgen05.cp.32x128b puts them into tensor memory (32 lanes, 4 columns of 4 bytes).
//              Bytes of rows past R and of blocks past K are zero.
//   row_scale  nvfp4: fp32 [R], a factor of the whole row.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace dmad {

constexpr int kFp4TileRows = 128;    // rows of a scale tile
constexpr int kFp4TileBlocks = 4;    // blocks of a scale tile
constexpr int kFp4TileBytes = 512;

__host__ __device__ constexpr int fp4_block(bool nv) { return nv ? 16 : 32; }

// Byte offset of the scale of (row, block) with `ktiles` scale tiles along K.
__host__ __device__ __forceinline__ int64_t fp4_scale_offset(int64_t row, int64_t block, int64_t ktiles) {
  return ((row >> 7) * ktiles + (block >> 2)) * kFp4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

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

// ---------------------------------------------------------------- conversions
// Eight floats -> eight e2m1 codes (v[0] in the low four bits): nearest, halves to the even code, 6 at most.
__device__ __forceinline__ uint32_t float8_to_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t3, %8, %7;\n\t"
      "mov.b32 %0, {t0, t1, t2, t3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight e2m1 codes -> floats (exact: every e2m1 number is an fp16 number).
__device__ __forceinline__ void e2m1x8_to_float8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, t2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// e4m3 code of a float >= 0 (nearest, halves to even, 448 at most) and its value (code 0x7f: NaN).
__device__ __forceinline__ uint32_t float_to_e4m3(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float e4m3_to_float(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}

// 2^(stored - 127) of a ue8m0 code (0xff: NaN).
__device__ __forceinline__ float ue8m0_to_float(uint32_t code) {
  return __uint_as_float(code == 0xffu ? 0x7fffffffu : code == 0u ? 0x00400000u : code << 23);
}

// ---------------------------------------------------------------- tensor core
// Instruction descriptor of the block-scaled 4-bit kinds (fp32 accumulator, both operands K-major e2m1):
//   [4,6) scale id of B; [7,10) A type (1 = e2m1); [10,12) B type; [17,23) N >> 3; bit 23 scale type
//   (0 = ue4m3, 1 = ue8m0); [27,29) M >> 7; [29,31) scale id of A; bit 31 K (0 = 64).
// The scale id is the byte of the 32-bit scale word at which the instruction's scales begin.
__host__ __device__ constexpr uint32_t idesc_fp4(bool nv, int M, int N, int scale_id) {
  return ((uint32_t)scale_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((nv ? 0u : 1u) << 23) |
         ((uint32_t)(M >> 7) << 27) | ((uint32_t)scale_id << 29);
}

// D[tmem] (+)= (A * scale_a)[smem] (B * scale_b)[smem]^T over 64 columns of K.  CG = 2: issued by one thread of a CTA
// pair for both, A's and D's rows split over the two CTAs and B's rows loaded half by each; every address is the
// same in both.
template <bool NV, int CG>
__device__ __forceinline__ void mma_fp4_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
#define DMAD_FP4_MMA(GROUP, KIND)                                                                                     \
  asm volatile("{\n\t.reg .pred p;\n\t"                                                                              \
               "setp.ne.b32 p, %6, 0;\n\t"                                                                           \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem), \
               "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)                   \
               : "memory")
  if constexpr (NV && CG == 1) DMAD_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (NV) DMAD_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (CG == 1) DMAD_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  else DMAD_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
#undef DMAD_FP4_MMA
}

// Descriptor of an unswizzled scale tile: 32 rows of 16 bytes, eight-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

// One scale tile (512 bytes) -> four columns of tensor memory, in each of the four lane quarters.  CG = 2: in both
// CTAs of the pair, each from its own shared memory.
template <int CG>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

}  // namespace dmad
