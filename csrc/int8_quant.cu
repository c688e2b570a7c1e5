// Quantisation of rows to 8-bit integers and back (int8.cuh has the layout and the formulas).
//
// The kernels read each element once and are bound by HBM.  A thread takes units of 16 columns (one 32-byte load of 16-bit
// elements, one 16-byte store of codes); a row with one scale is held by one block in registers between its maximum and the
// encoding (up to 32768 columns of 16 bits, 16384 of 32; longer rows are read twice).  Rows that do not start on 32
// bytes are read, and written back, in the aligned pieces around a unit (row_units.cuh).
// Measured at 37966 x 5120 bf16 (583 MB coded, 583 MB read back): blocks 88 to 91 us (6.4 to 6.6 TB/s), rows 137 to 140 us (4.2
// TB/s: six rows share an SM, each some 3 us from its first load over its maximum to its last store), inverse 88 to 91 us;
// fp32 blocks 138 to 140 us, rows 151 to 154 us (6.4 TB/s), inverse 146 to 148 us.  37966 x 5121: bf16 blocks 142 to 144 us,
// rows 194 to 197 us, inverse 142 to 155 us; fp32 183, 251, 161 to 179 us.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.cuh"
#include "int8_host.h"

namespace dmad {
namespace {

struct QuantParams {
  const void* x;
  int64_t ld;
  int R, K;
  int8_t* data;
  float* row_scale;
  uint8_t* exponents;
};

// blockDim = (threads of a row, rows); more than one warp a row means one row a block.
template <typename T, bool BLOCKS, bool ALIGNED, int UPT>
__global__ void __launch_bounds__(512, sizeof(T) == 4 || UPT > 2 ? 1 : 2) int8_quant_kernel(QuantParams p) {
  __shared__ uint32_t red[16];
  launch_dependents();  // a product that reads the codes may set itself up meanwhile (it waits for this grid's end)
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int TX = blockDim.x, lane = threadIdx.x & 31;
  const bool live = row < p.R;
  const int K = live ? p.K : 0;
  const int row_bytes = (int)int8_row_bytes(p.K);
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  int8_t* out = p.data + row * row_bytes;
  const int chunks = (row_bytes / 16 + TX * UPT - 1) / (TX * UPT);
  Unit<T> v[UPT];
  auto column = [&](int c, int i) { return (int)(threadIdx.x + (c * UPT + i) * TX) * 16; };  // first one of unit i
  auto load = [&](int c) {
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if constexpr (ALIGNED) v[i] = load_unit<T, true>(xr, column(c, i), K);
      else v[i] = load_unit_anywhere<T>(xr, column(c, i), K);
    }
  };
  auto store = [&](int col, const uint32_t (&codes)[4]) {
    if (live && col < row_bytes) *reinterpret_cast<uint4*>(out + col) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  };
  if constexpr (BLOCKS) {
    const int nb = row_bytes / kInt8Block;
    uint8_t* er = p.exponents + row * nb;
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int col = column(c, i);
        uint32_t codes[4];
        uint32_t amax = absmax_bits(v[i]);  // a block is two lanes' units
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        const uint32_t e = int8_block_code(amax);
        int8_encode_block(v[i], e, codes);
        if (live && (lane & 1) == 0 && col < row_bytes) er[col / kInt8Block] = (uint8_t)e;
        store(col, codes);
      }
    }
  } else {
    uint32_t m = 0;
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < UPT; ++i) m = max(m, absmax_bits(v[i]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (TX > 32) {
      if (lane == 0) red[threadIdx.x >> 5] = m;
      __syncthreads();
      m = __reduce_max_sync(0xffffffffu, lane < (TX >> 5) ? red[lane] : 0u);
    }
    const bool bad = m >= kInfBits;
    float inv;
    const float s = int8_row_scale(m, inv);
    if (threadIdx.x == 0 && live) p.row_scale[row] = s;
    for (int c = 0; c < chunks; ++c) {
      if (chunks > 1) load(c);
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        uint32_t codes[4] = {0u, 0u, 0u, 0u};
        if (!bad) int8_encode_row(v[i], s, inv, codes);
        store(column(c, i), codes);
      }
    }
  }
}

template <typename T, bool BLOCKS, bool ALIGNED>
void launch_quant(const QuantParams& p, cudaStream_t stream) {
  const int units = (int)(int8_row_bytes(p.K) / 16);
  constexpr int UPT = sizeof(T) == 4 ? 2 : 4;
  auto go = [&](auto upt) {
    constexpr int U = decltype(upt)::value;
    const int tx = std::min(512, ((units + U - 1) / U + 31) / 32 * 32), ty = tx == 32 ? 4 : 1;
    int8_quant_kernel<T, BLOCKS, ALIGNED, U><<<(unsigned)(((int64_t)p.R + ty - 1) / ty), dim3(tx, ty), 0, stream>>>(p);
  };
  // Two units a thread keep the rows of up to 16384 columns in one block of 512 threads.  (37966 x 5120 bf16, one scale a
  // row: 137 to 140 us; one unit a thread in 42 registers 217 us, four in 64, which spill, 168 us.)
  if constexpr (BLOCKS || UPT == 2) {
    go(std::integral_constant<int, 2>{});
  } else {
    if (units <= 1024) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, UPT>{});
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T>
void quant_typed(const QuantParams& p, cudaStream_t stream) {
  const bool aligned = p.K % 16 == 0 && (p.ld * sizeof(T)) % 32 == 0 && reinterpret_cast<uintptr_t>(p.x) % 32 == 0;
  if (p.exponents != nullptr) aligned ? launch_quant<T, true, true>(p, stream) : launch_quant<T, true, false>(p, stream);
  else aligned ? launch_quant<T, false, true>(p, stream) : launch_quant<T, false, false>(p, stream);
}

// ---------------------------------------------------------------- and back
template <typename O>
__device__ __forceinline__ uint32_t pack_pair(uint64_t v) {
  const float2 f = f2_split(v);
  if constexpr (std::is_same_v<O, __nv_bfloat16>) return f2_to_bf16x2(f.x, f.y);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename O, bool BLOCKS, bool ALIGNED>
__global__ void __launch_bounds__(256) int8_dequant_kernel(const int8_t* __restrict__ data, const float* __restrict__ row_scale,
                                                           const uint8_t* __restrict__ exponents, O* __restrict__ out, int64_t ld,
                                                           int R, int K) {
  __shared__ uint32_t turn[!ALIGNED && sizeof(O) == 4 ? 8 : 1][!ALIGNED && sizeof(O) == 4 ? 32 * 17 : 1];
  launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= R) return;  // whole warps
  const int row_bytes = (int)int8_row_bytes(K), nb = row_bytes / kInt8Block;
  const int8_t* dr = data + row * row_bytes;
  O* orow = out + row * ld;
  float s = BLOCKS ? 1.f : row_scale[row];
  const int lane = threadIdx.x & 31;
  // whole warps stay together
  for (int first = (threadIdx.x - lane) * 16; first < K; first += blockDim.x * 16) {
    const int c = first + lane * 16;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (c < K) {
      w = __ldg(reinterpret_cast<const uint4*>(dr + c));
      if constexpr (BLOCKS) s = int8_block_scale(__ldg(exponents + row * nb + c / kInt8Block));
    }
    const uint64_t s2 = f2(s, s);
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(O) == 4) {
      uint32_t o[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint64_t lo, hi;
        bytes_to_float(q[i], lo, hi);
        const float2 a = f2_split(f2_mul(lo, s2)), b = f2_split(f2_mul(hi, s2));
        o[4 * i] = __float_as_uint(a.x);
        o[4 * i + 1] = __float_as_uint(a.y);
        o[4 * i + 2] = __float_as_uint(b.x);
        o[4 * i + 3] = __float_as_uint(b.y);
      }
      if constexpr (ALIGNED) {  // K is a multiple of 16
        if (c < K) {
          st256(orow + c, o);
          st256(orow + c + 8, o + 8);
        }
      } else {  // through shared memory, in runs of the warp's lanes
        uint32_t* t = turn[threadIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5)];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) t[lane * 17 + i] = o[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int e = i * 32 + lane;
          if (first + e < K) reinterpret_cast<uint32_t*>(orow)[first + e] = t[(e >> 4) * 17 + (e & 15)];
        }
      }
    } else {
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint64_t lo, hi;
        bytes_to_float(q[i], lo, hi);
        o[2 * i] = pack_pair<O>(f2_mul(lo, s2));
        o[2 * i + 1] = pack_pair<O>(f2_mul(hi, s2));
      }
      if constexpr (ALIGNED) {
        if (c < K) st256(orow + c, o);
      } else {
        store_unit_anywhere(reinterpret_cast<uint16_t*>(orow), c, K, o);
      }
    }
  }
}

template <typename O, bool BLOCKS>
void launch_dequant(const Int8Matrix& q, void* out, int64_t ld, cudaStream_t stream) {
  const int R = (int)q.rows, K = (int)q.cols, units = (K + 15) / 16;
  const dim3 block = row_block(units);
  const unsigned grid = (unsigned)(((int64_t)R + block.y - 1) / block.y);
  const bool aligned = K % 16 == 0 && (ld * sizeof(O)) % 32 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  O* o = static_cast<O*>(out);
  if (aligned)
    int8_dequant_kernel<O, BLOCKS, true><<<grid, block, 0, stream>>>(q.data, q.row_scale, q.exponents, o, ld, R, K);
  else
    int8_dequant_kernel<O, BLOCKS, false><<<grid, block, 0, stream>>>(q.data, q.row_scale, q.exponents, o, ld, R, K);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

Int8Matrix int8_matrix(const at::Tensor& data, const at::Tensor& scale, int64_t rows, int64_t cols, bool blocks,
                       const at::Device& device, const char* name) {
  Int8Matrix m{nullptr, nullptr, nullptr, rows, cols};
  const std::string who(name);
  DMAD_VALUE_CHECK(cols >= 1 && cols <= (1 << 24) && rows >= 0 && rows <= INT32_MAX - 256, who + ": sizes out of range");
  DMAD_VALUE_CHECK(data.scalar_type() == at::kChar && data.dim() == 2 && data.size(0) == rows &&
                       data.size(1) == m.row_bytes() && data.is_contiguous(),
                   who + ".data must be contiguous int8 (" + num(rows) + ", " + num(m.row_bytes()) + "), got " +
                       shape_text(data));
  if (blocks) {
    DMAD_VALUE_CHECK(scale.scalar_type() == at::kByte && scale.dim() == 2 && scale.size(0) == rows &&
                         scale.size(1) == m.blocks() && scale.is_contiguous(),
                     who + ".scale must be contiguous uint8 (" + num(rows) + ", " + num(m.blocks()) + "), got " +
                         shape_text(scale));
  } else {
    DMAD_VALUE_CHECK(scale.scalar_type() == at::kFloat && scale.dim() == 1 && scale.size(0) == rows && scale.is_contiguous(),
                     who + ".scale must be contiguous fp32 (" + num(rows) + ",), got " + shape_text(scale));
  }
  DMAD_VALUE_CHECK(data.device() == device && scale.device() == device, who + ": data and scale must be on the device of x");
  m.data = reinterpret_cast<int8_t*>(data.data_ptr());
  if (blocks) m.exponents = scale.data_ptr<uint8_t>();
  else m.row_scale = scale.data_ptr<float>();
  DMAD_VALUE_CHECK(reinterpret_cast<uintptr_t>(m.data) % 16 == 0, who + ".data must start on 16 bytes");
  return m;
}

at::Tensor int8_rows(const at::Tensor& x, const char* name) {
  DMAD_VALUE_CHECK(x.dim() >= 1 && x.size(-1) >= 1, std::string(name) + ": the last dimension must hold at least one "
                                                                        "column, got " + shape_text(x));
  const int64_t K = x.size(-1);
  const at::Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  DMAD_VALUE_CHECK(K <= (1 << 24) && r.size(0) <= INT32_MAX - 256, std::string(name) + ": sizes out of range");
  return r.stride(1) == 1 || K == 1 ? r : r.contiguous();
}

void int8_quantize_launch(const at::Tensor& x, const Int8Matrix& q, cudaStream_t stream) {
  if (q.rows == 0) return;
  QuantParams p{x.data_ptr(), x.stride(0), (int)q.rows, (int)q.cols, q.data, q.row_scale, q.exponents};
  if (x.scalar_type() == at::kBFloat16) quant_typed<__nv_bfloat16>(p, stream);
  else if (x.scalar_type() == at::kHalf) quant_typed<__half>(p, stream);
  else quant_typed<float>(p, stream);
}

void int8_dequantize_launch(const Int8Matrix& q, const at::Tensor& out, cudaStream_t stream) {
  if (q.rows == 0) return;
  auto go = [&](auto tag) {
    using O = decltype(tag);
    if (q.exponents != nullptr) launch_dequant<O, true>(q, out.data_ptr(), out.stride(0), stream);
    else launch_dequant<O, false>(q, out.data_ptr(), out.stride(0), stream);
  };
  if (out.scalar_type() == at::kBFloat16) go(__nv_bfloat16{});
  else if (out.scalar_type() == at::kHalf) go(__half{});
  else go(float{});
}

// (data, scale) of x [..., K] (bf16, fp16 or fp32 on CUDA), with one scale a row or in blocks of 32 columns.
std::tuple<at::Tensor, at::Tensor> int8_quantize(const at::Tensor& x, bool blocks) {
  DMAD_VALUE_CHECK(x.is_cuda() && is_float_type(x.scalar_type()), "quantize_int8: x must be bf16, fp16 or fp32 on CUDA");
  c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor x2 = int8_rows(x, "quantize_int8");
  Int8Matrix q{nullptr, nullptr, nullptr, x2.size(0), x2.size(1)};
  const auto plain = x.options().requires_grad(false);
  at::Tensor data = at::empty({q.rows, q.row_bytes()}, plain.dtype(at::kChar));
  at::Tensor scale = blocks ? at::empty({q.rows, q.blocks()}, plain.dtype(at::kByte)) : at::empty({q.rows}, plain.dtype(at::kFloat));
  q.data = reinterpret_cast<int8_t*>(data.data_ptr());
  if (blocks) q.exponents = scale.data_ptr<uint8_t>();
  else q.row_scale = scale.data_ptr<float>();
  int8_quantize_launch(x2, q, at::cuda::getCurrentCUDAStream());
  return {data, scale};
}

// The values [R, K] that the codes stand for, rounded to bf16 (0), fp16 (1) or fp32 (2).
at::Tensor int8_dequantize(const at::Tensor& data, const at::Tensor& scale, int64_t R, int64_t K, bool blocks, int64_t type) {
  const Int8Matrix q = int8_matrix(data, scale, R, K, blocks, data.device(), "dequantize_int8: q");
  DMAD_VALUE_CHECK(data.is_cuda(), "dequantize_int8: the native kernel takes CUDA tensors");
  c10::cuda::CUDAGuard guard(data.device());
  at::Tensor out = at::empty({R, K}, data.options().dtype(type == 0 ? at::kBFloat16 : type == 1 ? at::kHalf : at::kFloat));
  int8_dequantize_launch(q, out, at::cuda::getCurrentCUDAStream());
  return out;
}

}  // namespace dmad
