// Quantisation of rows to block-scaled 4-bit floating point (e2m1) and back.
//
//   mxfp4:  s_b = 2^(floor(log2 max_b |x|) - 2),                       code = e2m1(x / s_b)
//   nvfp4:  g_r = the smallest 2^p with max_r |x| <= 6 * 448 * 2^p,
//           s_b = e4m3(max_b |x| / (6 g_r)),                           code = e2m1(x / (s_b g_r))
//
// (e2m1 and e4m3 round to nearest with halves to the even code; e2m1 saturates at 6, and what rounds to zero has code
// 0 whatever its sign.)  A block that holds an
// infinity or a NaN gets the scale code NaN, so all its values read back as NaN; such blocks do not count
// in g_r.  Scales are exact powers of two or quotients rounded once, so a code depends on nothing but the
// numbers: the CPU restatement gives the same bytes.
//
// The kernel reads each element once and is bound by HBM.  A thread takes units of 16 columns (one 32-byte
// load of 16-bit elements, one 8-byte store of codes); a row is held by one block in registers between the
// row maximum and the encoding, so nvfp4's two levels cost no second read while the row fits (32768 columns;
// longer rows are read twice).
// Measured at 37966 x 5120 bf16: nvfp4 quantiser 105 us (4.7 TB/s; bound by its instructions, some 230 for a thread's 16
// columns, which take 80 % of the issue slots; with 64 registers a thread 110 us, the bound to 40 for a third block of 512
// threads costs 96 bytes of spills; with IEEE divisions 127 us; one unit a thread instead of two 123 us), mxfp4 91 us (5.4
// TB/s), fp32 nvfp4 251 us (3.5 TB/s); inverse to bf16 82 us (6.1 TB/s).  Rows off 32 bytes are loaded by elements, one
// sector a lane: 37966 x 5121 248 us.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.cuh"
#include "fp4_host.h"
#include "sm100.cuh"

namespace dmad {
namespace {

constexpr uint32_t kInfBits = 0x7f800000u;

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

// The smallest power of two g with amax <= 6 * 448 * g (6 * 448 = 1.3125 * 2^11), 1 for amax = 0.
__device__ __forceinline__ float row_scale_of(uint32_t amax_bits) {
  if (amax_bits == 0u) return 1.f;
  int e = (int)(amax_bits >> 23) - 127 - 11 + ((amax_bits & 0x7fffffu) > 0x280000u ? 1 : 0);
  e = max(e, -126);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Eight codes with those of -0 made +0.
__device__ __forceinline__ uint32_t unsigned_zeros(uint32_t w) {
  const uint32_t some = (w | (w >> 1) | (w >> 2)) & 0x11111111u;  // codes that are not zero
  return w & (0x77777777u | (some << 3));
}

// Codes of 16 values x * m of 16-bit elements x.  Rounded to steps of 2^-15 first, by adding and subtracting 384: x m
// differs from a border b of two codes by 2^-11 b or more unless x over the scale is b, and where m is a rounded
// reciprocal it is off by no more than 2^-20; so the step moves such a product onto b and no other onto it.
template <typename T>
__device__ __forceinline__ void encode16(const Unit<T>& u, float m, uint32_t (&out)[2]) {
  const uint64_t m2 = f2(m, m), c = f2(384.f, 384.f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = f2_split(f2_sub(f2_fma(unit_pair(u, 4 * h + i), m2, c), c));
      y[2 * i] = v.x;
      y[2 * i + 1] = v.y;
    }
    out[h] = unsigned_zeros(float8_to_e2m1x8(y));
  }
}

// The same for fp32 elements, given the values.
__device__ __forceinline__ void encode32(const float (&v)[16], uint32_t (&out)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = v[8 * h + i];
    out[h] = unsigned_zeros(float8_to_e2m1x8(y));
  }
}

// Codes of one unit for nvfp4; returns the block's scale code.
template <typename T>
__device__ __forceinline__ uint32_t encode_nv(const Unit<T>& u, uint32_t amax, float ginv, uint32_t (&out)[2]) {
  if (amax >= kInfBits) {
    out[0] = out[1] = 0u;
    return 0x7fu;
  }
  const float top = __uint_as_float(amax) * ginv;
  if constexpr (sizeof(T) == 4) {
    const uint32_t code = float_to_e4m3(__fdiv_rn(top, 6.f));
    const float s = e4m3_to_float(code);
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = s > 0.f ? __fdiv_rn(__uint_as_float(u.w[i]) * ginv, s) : 0.f;
    encode32(v, out);
    return code;
  } else {
    // top / 6 by the rounded 1 / 6, then rounded to 17 bits: as above, that puts what is half-way between two e4m3
    // numbers (with an 11-bit top) back there and moves nothing else across
    const uint32_t q = (__float_as_uint(top * (1.f / 6.f)) + 0x40u) & ~0x7fu;
    const uint32_t code = float_to_e4m3(__uint_as_float(q));
    const float s = e4m3_to_float(code);
    float r;  // 1 / s to within 2^-23; 0 for a block without a scale
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    r = s > 0.f ? r : 0.f;
    if (ginv > 0x1p100f) {  // a row of tiny numbers: ginv r could overflow
      Unit<float> big;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 x = f2_split(unit_pair(u, i));
        big.w[2 * i] = __float_as_uint(x.x * ginv);
        big.w[2 * i + 1] = __float_as_uint(x.y * ginv);
      }
      encode16(big, r, out);
    } else {
      encode16(u, ginv * r, out);
    }
    return code;
  }
}

// Codes of one unit for mxfp4 with the block's (two units') maximum; returns the scale code.
template <typename T>
__device__ __forceinline__ uint32_t encode_mx(const Unit<T>& u, uint32_t amax, uint32_t (&out)[2]) {
  if (amax >= kInfBits) {
    out[0] = out[1] = 0u;
    return 0xffu;
  }
  const uint32_t code = (uint32_t)max((int)(amax >> 23) - 2, 0);
  const float m = __uint_as_float((254u - code) << 23);  // 2^(127 - code)
  if constexpr (sizeof(T) == 4) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(u.w[i]) * m;
    encode32(v, out);
  } else {
    encode16(u, m, out);
  }
  return code;
}

struct QuantParams {
  const void* x;
  int64_t ld;
  int R, K;
  uint8_t* data;
  uint8_t* scales;
  float* row_scale;
  int row_bytes, ktiles;
};

// blockDim = (threads of a row, rows); more than one warp a row means one row a block.
template <typename T, bool NV, bool ALIGNED, int UPT>
__global__ void __launch_bounds__(512, sizeof(T) == 4 || UPT > 2 ? 1 : 3) quant_kernel(QuantParams p) {
  __shared__ uint32_t red[16];
  launch_dependents();  // a product that reads the codes may set itself up meanwhile (it waits for this grid's end)
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int TX = blockDim.x;
  const int units = p.ktiles * kFp4TileBlocks * (fp4_block(NV) / 16);
  const bool live = row < p.R;
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  const int chunks = (units + TX * UPT - 1) / (TX * UPT);
  Unit<T> v[UPT];
  uint32_t top[UPT];  // maxima of the units
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int u = threadIdx.x + (c * UPT + i) * TX;
      v[i] = load_unit<T, ALIGNED>(xr, u * 16, live ? p.K : 0);
    }
  };
  float ginv = 1.f;
  if constexpr (NV) {
    uint32_t m = 0;
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        top[i] = absmax_bits(v[i]);
        m = max(m, top[i] < kInfBits ? top[i] : 0u);
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (TX > 32) {
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
      __syncthreads();
      const int nw = TX >> 5;
      m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < nw ? red[threadIdx.x & 31] : 0u);
    }
    const float g = row_scale_of(m);
    ginv = __uint_as_float((254u << 23) - __float_as_uint(g));  // 1 / g of a power of two
    if (threadIdx.x == 0 && live) p.row_scale[row] = g;
  }
  // rows past R up to the scale tile's end have zero scales and no data
  const bool tile_row = row < ((int64_t)p.R + kFp4TileRows - 1) / kFp4TileRows * kFp4TileRows;
  for (int c = 0; c < chunks; ++c) {
    if (!NV || chunks > 1) {
      load(c);
#pragma unroll
      for (int i = 0; i < UPT; ++i) top[i] = absmax_bits(v[i]);
    }
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int u = threadIdx.x + (c * UPT + i) * TX;
      uint32_t amax = top[i];
      uint32_t codes[2], sc;
      if constexpr (NV) {
        sc = encode_nv(v[i], amax, ginv, codes);
      } else {
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        sc = encode_mx(v[i], amax, codes);
      }
      if (live && u * 8 < p.row_bytes)
        *reinterpret_cast<uint2*>(p.data + row * p.row_bytes + (int64_t)u * 8) = make_uint2(codes[0], codes[1]);
      // the four scales of a tile's row are one word, stored by the first of their lanes
      constexpr int STEP = fp4_block(NV) / 16;
      uint32_t word = sc;
      word |= __shfl_down_sync(0xffffffffu, sc, STEP) << 8;
      word |= __shfl_down_sync(0xffffffffu, sc, 2 * STEP) << 16;
      word |= __shfl_down_sync(0xffffffffu, sc, 3 * STEP) << 24;
      if (u % (4 * STEP) == 0 && u < units && tile_row)
        *reinterpret_cast<uint32_t*>(p.scales + fp4_scale_offset(row, u / STEP, p.ktiles)) = word;
    }
  }
}

template <typename T, bool NV, bool ALIGNED>
void launch_quant(const QuantParams& p, cudaStream_t stream) {
  const int units = p.ktiles * kFp4TileBlocks * (fp4_block(NV) / 16);
  const int64_t rows = ((int64_t)p.R + kFp4TileRows - 1) / kFp4TileRows * kFp4TileRows;
  constexpr int UPT = sizeof(T) == 4 ? 2 : 4;
  auto go = [&](auto upt) {
    constexpr int U = decltype(upt)::value;
    int tx = (units + U - 1) / U;
    tx = std::min(512, (tx + 31) / 32 * 32);
    const int ty = tx == 32 ? 4 : 1;
    quant_kernel<T, NV, ALIGNED, U><<<(unsigned)((rows + ty - 1) / ty), dim3(tx, ty), 0, stream>>>(p);
  };
  // two units a thread keep the rows of up to 16384 columns in one block of 512 threads
  if (units <= 1024) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, UPT>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T>
void quant_typed(const QuantParams& p, bool nv, cudaStream_t stream) {
  const bool aligned = p.K % 16 == 0 && (p.ld * sizeof(T)) % 32 == 0 && reinterpret_cast<uintptr_t>(p.x) % 32 == 0;
  if (nv) aligned ? launch_quant<T, true, true>(p, stream) : launch_quant<T, true, false>(p, stream);
  else aligned ? launch_quant<T, false, true>(p, stream) : launch_quant<T, false, false>(p, stream);
}

// ---------------------------------------------------------------- dequantisation
template <typename O, bool NV, bool ALIGNED>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* __restrict__ data, int row_bytes,
                                                      const uint8_t* __restrict__ scales, int ktiles,
                                                      const float* __restrict__ row_scale, O* __restrict__ out, int R,
                                                      int K) {
  // rows of out that are no multiples of 32 bytes leave through shared memory, a warp's 512 columns at a time
  __shared__ float turn[ALIGNED ? 1 : 8][ALIGNED ? 1 : 32 * 17];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= R) return;
  const float g = NV ? row_scale[row] : 1.f;
  O* orow = out + row * K;
  const int lane = threadIdx.x & 31;
  // whole warps stay together: a lane past the row works on its last unit
  for (int first = threadIdx.x - lane; first * 16 < K; first += blockDim.x) {
    const int u = min(first + lane, (K - 1) / 16);
    if (ALIGNED && first + lane != u) continue;
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(data + row * row_bytes + (int64_t)u * 8));
    const uint32_t sc = __ldg(scales + fp4_scale_offset(row, NV ? u : u >> 1, ktiles));
    const float s = NV ? e4m3_to_float(sc) * g : ue8m0_to_float(sc);
    float f[16];
    {
      float a[8], b[8];
      e2m1x8_to_float8(w.x, a);
      e2m1x8_to_float8(w.y, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = a[i] * s;
        f[8 + i] = b[i] * s;
      }
    }
    if constexpr (ALIGNED) {
      if constexpr (sizeof(O) == 4) {
        st256(orow + u * 16, reinterpret_cast<const uint32_t*>(f));
        st256(orow + u * 16 + 8, reinterpret_cast<const uint32_t*>(f) + 8);
      } else {
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (std::is_same_v<O, __nv_bfloat16>) {
            o[i] = f2_to_bf16x2(f[2 * i], f[2 * i + 1]);
          } else {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            o[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        st256(orow + u * 16, o);
      }
    } else {
      float* t = turn[(threadIdx.y * blockDim.x + threadIdx.x) >> 5];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) t[lane * 17 + i] = f[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = i * 32 + lane, c = first * 16 + e;
        const float v = t[(e >> 4) * 17 + (e & 15)];
        if (c < K) {
          if constexpr (sizeof(O) == 4) orow[c] = v;
          else if constexpr (std::is_same_v<O, __nv_bfloat16>) orow[c] = __float2bfloat16_rn(v);
          else orow[c] = __float2half_rn(v);
        }
      }
    }
  }
}

template <typename O, bool NV>
void launch_dequant(const Fp4Matrix& q, at::Tensor& out, cudaStream_t stream) {
  const int R = (int)q.rows, K = (int)q.cols, row_bytes = (int)q.row_bytes(), ktiles = (int)q.ktiles();
  const int units = (K + 15) / 16;
  const int tx = std::min(256, (units + 31) / 32 * 32), ty = 256 / tx;
  const unsigned grid = (unsigned)((R + ty - 1) / ty);
  const bool aligned = K % 16 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 32 == 0;
  O* o = reinterpret_cast<O*>(out.data_ptr());
  if (aligned)
    dequant_kernel<O, NV, true><<<grid, dim3(tx, ty), 0, stream>>>(q.data, row_bytes, q.scales, ktiles, q.row_scale, o, R, K);
  else
    dequant_kernel<O, NV, false><<<grid, dim3(tx, ty), 0, stream>>>(q.data, row_bytes, q.scales, ktiles, q.row_scale, o, R, K);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

Fp4Matrix fp4_matrix(const at::Tensor& data, const at::Tensor& scales, const c10::optional<at::Tensor>& row_scale,
                     int64_t rows, int64_t cols, bool nv, const at::Device& device, const char* name) {
  Fp4Matrix m{nullptr, nullptr, nullptr, rows, cols, nv};
  const std::string who(name);
  DMAD_VALUE_CHECK(cols >= 1 && cols <= (1 << 24) && rows >= 0 && rows <= INT32_MAX - 256, who + ": sizes out of range");
  DMAD_VALUE_CHECK(data.scalar_type() == at::kByte && data.dim() == 2 && data.size(0) == rows &&
                       data.size(1) == m.row_bytes() && data.is_contiguous(),
                   who + ".data must be contiguous uint8 (" + num(rows) + ", " + num(m.row_bytes()) + "), got " +
                       shape_text(data));
  DMAD_VALUE_CHECK(scales.scalar_type() == at::kByte && scales.dim() == 3 && scales.size(0) == m.row_tiles() &&
                       scales.size(1) == m.ktiles() && scales.size(2) == kFp4TileBytes && scales.is_contiguous(),
                   who + ".scales must be contiguous uint8 (" + num(m.row_tiles()) + ", " + num(m.ktiles()) +
                       ", 512), got " + shape_text(scales));
  const bool has_rs = row_scale.has_value() && row_scale->defined();
  DMAD_VALUE_CHECK(nv == has_rs, who + ": nvfp4 has a row_scale and mxfp4 has none");
  DMAD_VALUE_CHECK(!nv || (row_scale->scalar_type() == at::kFloat && row_scale->dim() == 1 &&
                           row_scale->size(0) == rows && row_scale->is_contiguous()),
                   who + ".row_scale must be contiguous fp32 (" + num(rows) + ",)");
  DMAD_VALUE_CHECK(data.device() == device && scales.device() == device && (!nv || row_scale->device() == device),
                   who + ": all tensors must be on one device");
  m.data = data.data_ptr<uint8_t>();
  m.scales = scales.data_ptr<uint8_t>();
  m.row_scale = nv ? row_scale->data_ptr<float>() : nullptr;
  DMAD_VALUE_CHECK(reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && reinterpret_cast<uintptr_t>(m.scales) % 16 == 0,
                   who + ": data and scales must start on 16 bytes");
  return m;
}

void fp4_quantize_launch(const at::Tensor& x, const Fp4Matrix& q, cudaStream_t stream) {
  if (q.rows == 0) return;
  QuantParams p;
  p.x = x.data_ptr();
  p.ld = x.stride(0);
  p.R = (int)q.rows;
  p.K = (int)q.cols;
  p.data = q.data;
  p.scales = q.scales;
  p.row_scale = q.row_scale;
  p.row_bytes = (int)q.row_bytes();
  p.ktiles = (int)q.ktiles();
  if (x.scalar_type() == at::kBFloat16) quant_typed<__nv_bfloat16>(p, q.nv, stream);
  else if (x.scalar_type() == at::kHalf) quant_typed<__half>(p, q.nv, stream);
  else quant_typed<float>(p, q.nv, stream);
}

// x [..., K] as a matrix [R, K] with contiguous columns.
at::Tensor fp4_rows(const at::Tensor& x, const char* name) {
  DMAD_VALUE_CHECK(x.dim() >= 1 && x.size(-1) >= 1, std::string(name) + ": the last dimension must hold at least one "
                                                                        "column, got " + shape_text(x));
  const int64_t K = x.size(-1);
  at::Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  return r.stride(1) == 1 || K == 1 ? r : r.contiguous();
}

// (data, scales, row_scale) of x [..., K] (bf16, fp16 or fp32 on CUDA).
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>> fp4_quantize(const at::Tensor& x, bool nv) {
  DMAD_VALUE_CHECK(x.is_cuda() && is_float_type(x.scalar_type()), "quantize_fp4: x must be bf16, fp16 or fp32 on CUDA");
  const at::Tensor x2 = fp4_rows(x, "quantize_fp4");
  Fp4Matrix q{nullptr, nullptr, nullptr, x2.size(0), x2.size(1), nv};
  DMAD_VALUE_CHECK(q.cols <= (1 << 24) && q.rows <= INT32_MAX - 256, "quantize_fp4: sizes out of range");
  c10::cuda::CUDAGuard guard(x.device());
  const auto bytes = x.options().dtype(at::kByte).requires_grad(false);
  at::Tensor data = at::empty({q.rows, q.row_bytes()}, bytes);
  at::Tensor scales = at::empty({q.row_tiles(), q.ktiles(), kFp4TileBytes}, bytes);
  c10::optional<at::Tensor> rs;
  if (nv) rs = at::empty({q.rows}, bytes.dtype(at::kFloat));
  q.data = data.data_ptr<uint8_t>();
  q.scales = scales.data_ptr<uint8_t>();
  q.row_scale = nv ? rs->data_ptr<float>() : nullptr;
  fp4_quantize_launch(x2, q, at::cuda::getCurrentCUDAStream());
  return {data, scales, rs};
}

// The values [R, K] that the codes stand for, rounded to bf16 (0), fp16 (1) or fp32 (2).
at::Tensor fp4_dequantize(const at::Tensor& data, const at::Tensor& scales, c10::optional<at::Tensor> row_scale,
                          int64_t R, int64_t K, bool nv, int64_t type) {
  const Fp4Matrix q = fp4_matrix(data, scales, row_scale, R, K, nv, data.device(), "dequantize_fp4");
  DMAD_VALUE_CHECK(data.is_cuda(), "dequantize_fp4: the native kernel takes CUDA tensors");
  c10::cuda::CUDAGuard guard(data.device());
  at::Tensor out = at::empty({R, K}, data.options().dtype(type == 0 ? at::kBFloat16 : type == 1 ? at::kHalf : at::kFloat));
  if (R == 0) return out;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto tag) {
    using O = decltype(tag);
    nv ? launch_dequant<O, true>(q, out, stream) : launch_dequant<O, false>(q, out, stream);
  };
  if (type == 0) go(__nv_bfloat16{});
  else if (type == 1) go(__half{});
  else go(float{});
  return out;
}

}  // namespace dmad
