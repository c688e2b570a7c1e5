// A linear layer with an activation in front of it that keeps its input for the backward pass in 8 bits.
//
//   y = a W^T + bias,   a = act(x)                               x [R, F] (SwiGLU: [R, 2 F], value and gate), W [N, F]
//   kept: the codes of x in blocks of 32 columns (int8.cuh; a SwiGLU's halves each from their start), x' their values
//   dW = g^T act(x'),   dx = (g W) act'(x'),   db = sum g
//
//   gelu    v p with p = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)      (0.5 (1 + tanh u) = p)
//           derivative p + 2 v p (1 - p) u'
//   SwiGLU  v u p with p = 1 / (1 + exp(-u)); derivatives u p and v p (1 + u (1 - p))
//
// The products run on gemm_pair.cuh; operands that lie transposed are read MN-major where they are.  a is rounded to the
// operands' 16 bits, as the tensor core takes it; sums, activations and derivatives are fp32, rounded once.
//   forward     one pass over x writes a and the codes, then the product.  (Without an activation x itself is the operand.)
//   backward    the epilogue of g W reads the codes (1 byte an element) and writes dx and act(x') in one go: g W never
//               reaches memory and x' is decoded once for both; then g^T act(x').  Without an activation x' is decoded for
//               that product.
// Few output tiles: the K steps of a tile are spread over several pairs, whose fp32 parts are added in order by a second
// kernel, so that the sums are the same every time.
// Measured, forward and backward in short runs on several cards: 32760 x 1536 -> 4608 1.03 to 1.09 ms (1.28 to 1.35 PFLOP/s),
// 32760 x 8960 -> 1536 with GELU 2.17 to 2.30 ms, 37966 x 15360 -> 5120 with SwiGLU 13.2 to 15.9 ms (1.13 to 1.36 PFLOP/s); bound
// by the tensor core (1.55 PFLOP/s in the plain products, less as the power limit takes the clock) but for g W with few K
// steps, whose epilogue takes longer than its MMAs.  The coding pass: 32760 x 8960 GELU 230 us, 37966 x 15360
// SwiGLU 690 us (6.7 TB/s).
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "act8.h"
#include "common.cuh"
#include "gemm_pair.cuh"
#include "int8_host.h"

namespace dmad {
namespace {

// ---------------------------------------------------------------- activations
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + 2^z) of two numbers: 2^z of 2^128 and more is infinity, and the quotient 0.
__device__ __forceinline__ uint64_t logistic2(uint64_t z) {
  const float2 v = f2_split(z);
  const float2 d = f2_split(f2_add(f2(ex2_approx(v.x), ex2_approx(v.y)), f2(1.f, 1.f)));
  return f2(rcp_fast(d.x), rcp_fast(d.y));
}
__device__ __forceinline__ uint64_t both(float v) { return f2(v, v); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluC = 2.f * 0.7978845608028654f, kGeluA = -kGeluC * kLog2e, kGeluB = 0.044715f;

// Two elements at a time, in packed arithmetic: act(v), or act(v, u) of value and gate.
template <int ACT>
__device__ __forceinline__ uint64_t act_value(uint64_t v, uint64_t u) {
  if constexpr (ACT == kActGelu) {
    const uint64_t z = f2_mul(v, f2_fma(f2_mul(v, v), both(kGeluA * kGeluB), both(kGeluA)));  // -2 u log2(e)
    return f2_mul(v, logistic2(z));
  } else if constexpr (ACT == kActSwiglu) {
    return f2_mul(v, f2_mul(u, logistic2(f2_mul(u, both(-kLog2e)))));
  } else {
    return v;
  }
}

// act(x') and da act'(x'): dv, and for a SwiGLU du.
template <int ACT>
__device__ __forceinline__ void act_backward(uint64_t da, uint64_t v, uint64_t u, uint64_t& a, uint64_t& dv, uint64_t& du) {
  if constexpr (ACT == kActGelu) {
    // v v is bounded, so that slope stays finite where rest is 0: for |v| above 11, p is 0 or 1
    const float2 vv = f2_split(f2_mul(v, v));
    const uint64_t s = f2(fminf(vv.x, 1024.f), fminf(vv.y, 1024.f));
    const uint64_t p = logistic2(f2_mul(v, f2_fma(s, both(kGeluA * kGeluB), both(kGeluA))));
    a = f2_mul(v, p);
    const uint64_t rest = f2_sub(a, f2_mul(a, p)), slope = f2_fma(s, both(3.f * kGeluB * kGeluC), both(kGeluC));  // v p (1 - p), 2 u'
    dv = f2_mul(da, f2_fma(rest, slope, p));
    du = 0;
  } else if constexpr (ACT == kActSwiglu) {
    const uint64_t p = logistic2(f2_mul(u, both(-kLog2e))), up = f2_mul(u, p);
    a = f2_mul(v, up);
    dv = f2_mul(da, up);
    du = f2_mul(f2_mul(da, f2_add(f2_sub(up, f2_mul(up, p)), p)), v);  // (da v may be larger than fp32 where the slope is 0)
  } else {
    a = v;
    dv = da;
    du = 0;
  }
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack16x2(uint64_t v) {
  const float2 f = f2_split(v);
  return pack16<FP16>(f.x, f.y);
}

// Kept input: H = 2 for a SwiGLU (row r's halves are rows 2 r and 2 r + 1 of the codes), else 1.
struct Kept {
  int8_t* data;
  uint8_t* exponents;
};

// ---------------------------------------------------------------- forward pass over x
struct EncodeParams {
  const void* x;
  int64_t ld;
  int R, F;
  void* a;
  int64_t lda;
  Kept kept;  // data null: nothing is kept
};

template <typename T, int ACT, bool ALIGNED>
__global__ void __launch_bounds__(256) act_encode_kernel(EncodeParams p) {
  constexpr bool FP16 = std::is_same_v<T, __half>;
  constexpr int H = ACT == kActSwiglu ? 2 : 1;
  launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.R) return;  // whole warps
  const int lane = threadIdx.x & 31;
  const int row_bytes = (int)int8_row_bytes(p.F), nb = row_bytes / kInt8Block;
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  uint16_t* ar = static_cast<uint16_t*>(p.a) + row * p.lda;
  for (int first = threadIdx.x - lane; first * 16 < row_bytes; first += blockDim.x) {
    const int col = (first + lane) * 16;
    Unit<T> v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if constexpr (ALIGNED) v[h] = load_unit<T, true>(xr + h * p.F, col, p.F);
      else v[h] = load_unit_anywhere<T>(xr + h * p.F, col, p.F);
    }
    if (col < p.F) {  // (a's rows are padded to whole units)
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (ACT == kActNone) o[i] = v[0].w[i];
        else o[i] = pack16x2<FP16>(act_value<ACT>(unit_pair(v[0], i), unit_pair(v[H - 1], i)));
      }
      st256(ar + col, o);
    }
    if (p.kept.data == nullptr) continue;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint32_t amax = absmax_bits(v[h]);  // a block is two lanes' units
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      const uint32_t e = int8_block_code(amax);
      uint32_t codes[4];
      int8_encode_block(v[h], e, codes);
      if (col < row_bytes) {
        const int64_t r = row * H + h;
        *reinterpret_cast<uint4*>(p.kept.data + r * row_bytes + col) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        if ((lane & 1) == 0) p.kept.exponents[r * nb + col / kInt8Block] = (uint8_t)e;
      }
    }
  }
}

// act(x') [R, F] of the kept codes, for a backward pass without dx.  A thread takes four columns (a has room for them).
template <bool FP16, int ACT>
__global__ void __launch_bounds__(256) act_decode_kernel(Kept kept, uint16_t* a, int64_t lda, int R, int F) {
  constexpr int H = ACT == kActSwiglu ? 2 : 1;
  launch_dependents();
  const int row_bytes = (int)int8_row_bytes(F), nb = row_bytes / kInt8Block;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= R) return;
  for (int c = threadIdx.x * 4; c < F; c += blockDim.x * 4) {
    uint64_t v[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int64_t r = row * H + h;
      const float s = int8_block_scale(__ldg(kept.exponents + r * nb + c / kInt8Block));
      uint64_t lo, hi;
      bytes_to_float(__ldg(reinterpret_cast<const uint32_t*>(kept.data + r * row_bytes + c)), lo, hi);
      v[h][0] = f2_mul(lo, both(s));
      v[h][1] = f2_mul(hi, both(s));
    }
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) o[i] = pack16x2<FP16>(act_value<ACT>(v[0][i], v[H - 1][i]));
    *reinterpret_cast<uint2*>(a + row * lda + c) = make_uint2(o[0], o[1]);
  }
}

// ---------------------------------------------------------------- epilogues
// acc + bias -> 16 bits.
template <bool FP16>
struct BiasEpilogue {
  static constexpr int kStages = 6, kWarps = 8, kOutBytes = 2048;
  static constexpr bool kShared = true, kAhead = true;
  struct Args {
    CUtensorMap map;
    OutRows out;
    FloatRow bias;
  };
  const Args& a;
  const PairGemm& p;
  const EpiPlace at;
  int m0, n0;
  float next_bias;
  const float* col;

  __device__ __forceinline__ BiasEpilogue(const Args& a, const PairGemm& p, const EpiPlace& at) : a(a), p(p), at(at) {}
  __device__ __forceinline__ void fetch(int item) {
    int tm, tn;
    p.tile(item, tm, tn);
    next_bias = a.bias.at(min(tn * kPairN + at.thread, p.N - 1));
  }
  __device__ __forceinline__ void first(int item) { fetch(item); }
  __device__ __forceinline__ void begin(int item, int, int parity) {
    int tm, tn;
    p.tile(item, tm, tn);
    m0 = tm * kPairM + (int)at.rank * kPairHalf + at.wq * 32;
    n0 = tn * kPairN;
    float* mine = reinterpret_cast<float*>(at.col) + parity * kPairN;
    col = mine;
    mine[at.thread] = next_bias;
  }
  __device__ __forceinline__ void met(int next) {
    if (next >= 0) fetch(next);
  }
  __device__ __forceinline__ void chunk(int c, const uint32_t (&v)[32]) {
    const int nc = n0 + c * 32;
    if (nc >= p.N || m0 >= p.M) return;
    uint32_t o[16];
    const float4* f4 = reinterpret_cast<const float4*>(col + c * 32);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 f = f4[q];
      o[2 * q] = pack16<FP16>(__uint_as_float(v[4 * q]) + f.x, __uint_as_float(v[4 * q + 1]) + f.y);
      o[2 * q + 1] = pack16<FP16>(__uint_as_float(v[4 * q + 2]) + f.z, __uint_as_float(v[4 * q + 3]) + f.w);
    }
    if (at.lane == 0) tma_store_wait_read();
    __syncwarp();
    store_rows(a.out, &a.map, at.stage, m0, nc, o);
  }
};

// dx = acc act'(x') and act(x'), from the accumulator (g W) and the kept codes.  Some thirty instructions an element, with
// chains of dependent ones: sixteen warps, four a scheduler, and one copy of the code (eight warps with four unrolled
// chunks: 32760 x 1536 -> 8960 GELU 826 us, stalled on results and on the instruction cache).  A lane reads its row's 32
// codes of a chunk (one sector) while the chunk before is computed.  32760 x 1536 -> 8960: 740 to 762 us with the GELU's
// derivative, 880 to 919 us with the SwiGLU's, 638 to 653 us without any (on two cards); 37966 x 5120 -> 15360 (four times as
// many K steps a tile) is bound by the MMAs.
template <bool FP16, int ACT>
struct ActGradEpilogue {
  static constexpr int H = ACT == kActSwiglu ? 2 : 1;
  static constexpr int kStages = 6, kWarps = 16, kOutBytes = 2048;
  static constexpr bool kShared = false, kAhead = false;
  struct Args {
    CUtensorMap map_dx[H], map_a;
    OutRows dx[H], act;
    bool want_act;
    Kept kept;
  };
  struct Codes {
    uint4 lo, hi;
    uint32_t e;
  };
  const Args& a;
  const PairGemm& p;
  const EpiPlace at;
  int m0, n0;
  Codes next[H];

  __device__ __forceinline__ ActGradEpilogue(const Args& a, const PairGemm& p, const EpiPlace& at) : a(a), p(p), at(at) {}
  __device__ __forceinline__ void first(int) {}
  __device__ __forceinline__ void load(int c) {
    const int nc = n0 + c * 32, m = m0 + at.lane;
    const int row_bytes = (int)int8_row_bytes(p.N), nb = row_bytes / kInt8Block;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      next[h] = Codes{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0), 0u};
      if (m < p.M && nc < p.N && c < kPairN / 32) {
        const int64_t r = (int64_t)m * H + h;
        const uint4* d = reinterpret_cast<const uint4*>(a.kept.data + r * row_bytes + nc);
        next[h].lo = __ldg(d);
        next[h].hi = __ldg(d + 1);
        next[h].e = __ldg(a.kept.exponents + r * nb + nc / kInt8Block);
      }
    }
  }
  __device__ __forceinline__ void begin(int item, int, int) {
    int tm, tn;
    p.tile(item, tm, tn);
    m0 = tm * kPairM + (int)at.rank * kPairHalf + at.wq * 32;
    n0 = tn * kPairN;
    load(at.group);
  }
  __device__ __forceinline__ void chunk(int c, const uint32_t (&v)[32]) {
    const int nc = n0 + c * 32;
    Codes k[H];
#pragma unroll
    for (int h = 0; h < H; ++h) k[h] = next[h];
    load(c + kWarps / 4);
    if (nc >= p.N || m0 >= p.M) return;
    uint32_t od[H][16], oa[16];
    uint64_t s[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float f = int8_block_scale(k[h].e);
      s[h] = f2(f, f);
    }
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      uint64_t x[H][2];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint32_t bytes = w == 0 ? k[h].lo.x : w == 1 ? k[h].lo.y : w == 2 ? k[h].lo.z : w == 3 ? k[h].lo.w
                               : w == 4 ? k[h].hi.x : w == 5 ? k[h].hi.y : w == 6 ? k[h].hi.z : k[h].hi.w;
        uint64_t lo, hi;
        bytes_to_float(bytes, lo, hi);
        x[h][0] = f2_mul(lo, s[h]);
        x[h][1] = f2_mul(hi, s[h]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint64_t act, dv, du;
        const uint64_t da = f2(__uint_as_float(v[4 * w + 2 * j]), __uint_as_float(v[4 * w + 2 * j + 1]));
        act_backward<ACT>(da, x[0][j], x[H - 1][j], act, dv, du);
        oa[2 * w + j] = pack16x2<FP16>(act);
        od[0][2 * w + j] = pack16x2<FP16>(dv);
        if constexpr (H == 2) od[1][2 * w + j] = pack16x2<FP16>(du);
      }
    }
    auto store = [&](const OutRows& out, const CUtensorMap* map, const uint32_t (&o)[16]) {
      if (at.lane == 0) tma_store_wait_read();
      __syncwarp();
      store_rows(out, map, at.stage, m0, nc, o);
    };
#pragma unroll
    for (int h = 0; h < H; ++h) store(a.dx[h], &a.map_dx[h], od[h]);
    if (a.want_act) store(a.act, &a.map_a, oa);
  }
};

// ---------------------------------------------------------------- sums of parts
struct PartSum {
  const float* parts;
  PairGemm g;
  OutRows out[2];      // the result, or dx (of a SwiGLU: its halves)
  FloatRow bias;
  OutRows act;         // act(x'), if wanted
  bool want_act;
  Kept kept;
};

// Four columns a thread: the parts added in order, then what the epilogue of an undivided tile does.
template <bool FP16, int ACT>
__global__ void __launch_bounds__(kPartThreads) part_sum_kernel(const __grid_constant__ PartSum p) {
  constexpr int H = ACT == kActSwiglu ? 2 : 1;
  launch_dependents();
  wait_for_previous_grid();
  int m, n;
  int64_t at;
  if (!part_place(p.g, m, n, at)) return;
  float4 sum = *reinterpret_cast<const float4*>(p.parts + at);
  for (int s = 1; s < p.g.split; ++s) {
    const float4 f = *reinterpret_cast<const float4*>(p.parts + at + s * kPartStep);
    sum.x += f.x;
    sum.y += f.y;
    sum.z += f.z;
    sum.w += f.w;
  }
  float v[4] = {sum.x, sum.y, sum.z, sum.w};
  if constexpr (ACT == kActNone) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += p.bias.at(min(n + i, p.g.N - 1));
    store4<FP16>(p.out[0], m, n, v);
  } else {
    const int row_bytes = (int)int8_row_bytes(p.g.N), nb = row_bytes / kInt8Block;
    uint64_t x[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int64_t r = (int64_t)m * H + h;
      const float s = int8_block_scale(__ldg(p.kept.exponents + r * nb + n / kInt8Block));
      uint64_t lo, hi;
      bytes_to_float(__ldg(reinterpret_cast<const uint32_t*>(p.kept.data + r * row_bytes + n)), lo, hi);
      x[h][0] = f2_mul(lo, both(s));
      x[h][1] = f2_mul(hi, both(s));
    }
    float act[4], dv[4], du[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint64_t a2, v2, u2;
      act_backward<ACT>(f2(v[2 * j], v[2 * j + 1]), x[0][j], x[H - 1][j], a2, v2, u2);
      const float2 fa = f2_split(a2), fv = f2_split(v2), fu = f2_split(u2);
      act[2 * j] = fa.x, act[2 * j + 1] = fa.y;
      dv[2 * j] = fv.x, dv[2 * j + 1] = fv.y;
      du[2 * j] = fu.x, du[2 * j + 1] = fu.y;
    }
    store4<FP16>(p.out[0], m, n, dv);
    if constexpr (H == 2) store4<FP16>(p.out[1], m, n, du);
    if (p.want_act) store4<FP16>(p.act, m, n, act);
  }
}

// ---------------------------------------------------------------- sums of columns
// out[slice, n] = sum of rows slice * per .. of g: 256 columns a block, eight a lane, the block's warps on every eighth row.
template <bool FP16>
__global__ void __launch_bounds__(256) column_sum_kernel(const uint16_t* g, int64_t ld, int R, int N, int per, void* out, int type) {
  __shared__ float red[8][256];
  launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * 256 + lane * 8;
  const int r0 = blockIdx.y * per, r1 = min(R, r0 + per);
  float s[8] = {};
  if (n + 8 <= N) {
#pragma unroll 4
    for (int r = r0 + warp; r < r1; r += 8) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(g + (int64_t)r * ld + n));
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = FP16 ? __half22float2(*reinterpret_cast<const __half2*>(&q[i])) : unpack_bf16x2(q[i]);
        s[2 * i] += f.x;
        s[2 * i + 1] += f.y;
      }
    }
  } else {
    for (int r = r0 + warp; r < r1; r += 8)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) {
          const uint16_t w = g[(int64_t)r * ld + n + i];
          s[i] += FP16 ? __half2float(__ushort_as_half(w)) : __uint_as_float((uint32_t)w << 16);
        }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) red[warp][lane * 8 + i] = s[i];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += red[w][threadIdx.x];
  const int64_t to = (int64_t)blockIdx.y * N + c;
  if (type == 0) static_cast<float*>(out)[to] = t;
  else if (type == 1) static_cast<__nv_bfloat16*>(out)[to] = __float2bfloat16_rn(t);
  else static_cast<__half*>(out)[to] = __float2half_rn(t);
}

__global__ void __launch_bounds__(256) slice_sum_kernel(const float* parts, int slices, int N, void* out, int type) {
  launch_dependents();
  wait_for_previous_grid();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float t = 0.f;
  for (int s = 0; s < slices; ++s) t += parts[(int64_t)s * N + c];
  if (type == 0) static_cast<float*>(out)[c] = t;
  else if (type == 1) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(t);
  else static_cast<__half*>(out)[c] = __float2half_rn(t);
}

int type_index(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }

at::Tensor column_sum(const at::Tensor& g, at::ScalarType type, cudaStream_t stream) {
  const int R = (int)g.size(0), N = (int)g.size(1), nb = (N + 255) / 256, device = g.get_device();
  at::Tensor out = at::empty({N}, g.options().dtype(type));
  // slices for eight blocks an SM, of 64 rows at least
  const int slices = std::max(1, std::min(8 * sm_count(device) / nb, R / 64)), per = (R + slices - 1) / slices;
  at::Tensor parts = slices > 1 ? at::empty({slices, N}, g.options().dtype(at::kFloat)) : out;
  void* to = parts.data_ptr();
  const int first = slices > 1 ? 0 : type_index(type);
  const uint16_t* gp = static_cast<const uint16_t*>(g.data_ptr());
  if (g.scalar_type() == at::kHalf)
    column_sum_kernel<true><<<dim3(nb, slices), 256, 0, stream>>>(gp, g.stride(0), R, N, per, to, first);
  else
    column_sum_kernel<false><<<dim3(nb, slices), 256, 0, stream>>>(gp, g.stride(0), R, N, per, to, first);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (slices > 1)
    launch_overlapping(slice_sum_kernel, dim3(nb), dim3(256), 0, stream, true, (const float*)parts.data_ptr<float>(), slices, N,
                       out.data_ptr(), type_index(type));
  return out;
}

// ---------------------------------------------------------------- products
int halves(int64_t act) { return act == kActSwiglu ? 2 : 1; }

Kept kept_of(const at::Tensor& data, const at::Tensor& exponents) {
  return Kept{reinterpret_cast<int8_t*>(data.data_ptr()), exponents.data_ptr<uint8_t>()};
}

// act(x) [R, F] (no activation: a copy of x) with rows on 32 bytes, and the codes of x where they are kept.
at::Tensor encode(const at::Tensor& x2, int64_t F, int64_t act, const Kept& kept, cudaStream_t stream) {
  const int64_t R = x2.size(0), lda = (F + 15) / 16 * 16;
  at::Tensor a = at::empty({R, lda}, x2.options().requires_grad(false));
  if (R > 0) {
    const EncodeParams p{x2.data_ptr(), x2.stride(0), (int)R, (int)F, a.data_ptr(), lda, kept};
    const bool aligned = F % 16 == 0 && x2.stride(0) % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 32 == 0;
    const dim3 block = row_block(int8_row_bytes(F) / 16);
    const unsigned grid = (unsigned)((R + block.y - 1) / block.y);
    auto go = [&](auto tag, auto which) {
      using T = decltype(tag);
      constexpr int ACT = decltype(which)::value;
      if (aligned) act_encode_kernel<T, ACT, true><<<grid, block, 0, stream>>>(p);
      else act_encode_kernel<T, ACT, false><<<grid, block, 0, stream>>>(p);
    };
    auto typed = [&](auto tag) {
      if (act == kActNone) go(tag, std::integral_constant<int, kActNone>{});
      else if (act == kActGelu) go(tag, std::integral_constant<int, kActGelu>{});
      else go(tag, std::integral_constant<int, kActSwiglu>{});
    };
    if (x2.scalar_type() == at::kHalf) typed(__half{});
    else typed(__nv_bfloat16{});
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return a.narrow(1, 0, F);
}

// Whether TMA can read t's rows: contiguous columns, rows on 16 bytes.
bool tma_readable(const at::Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// Such rows: t, or a copy where it is laid out otherwise.
at::Tensor tma_rows(const at::Tensor& t, cudaStream_t stream) {
  if (tma_readable(t)) return t;
  if (t.stride(1) == 1) return encode(t, t.size(1), kActNone, Kept{nullptr, nullptr}, stream);
  at::Tensor p = at::empty({t.size(0), (t.size(1) + 7) / 8 * 8}, t.options().requires_grad(false)).narrow(1, 0, t.size(1));
  p.copy_(t);
  return p;
}

struct Operand {  // [rows, K], or stored [K, rows]
  const at::Tensor& t;
  bool mn;
  int64_t rows() const { return t.size(mn ? 1 : 0); }
  int64_t K() const { return t.size(mn ? 0 : 1); }
  CUtensorMap map() const { return operand_map(t.data_ptr(), rows(), K(), t.stride(0), 2, mn); }
};

// What becomes of the product (early: as PairGemm has it): out = acc + bias, or (act) out = acc act'(x') and act(x').
struct Result {
  OutRows out[2];
  FloatRow bias{nullptr, 0};
  int act = kActNone;
  Kept kept{nullptr, nullptr};
  OutRows value{};
  bool want_value = false;
  int early = 0;
  bool b_old = false;
};

template <bool FP16, int ACT>
void product_typed(const Operand& A, const Operand& B, const Result& r, int device, cudaStream_t stream) {
  constexpr Mma KIND = FP16 ? Mma::kF16 : Mma::kBf16;
  const int64_t M = A.rows(), N = B.rows(), K = A.K();
  PairGemm p = pair_gemm(M, N, K, 2, A.mn, B.mn, device);
  p.early = r.early;
  p.b_old = r.b_old ? 1 : 0;
  const at::Tensor parts = part_memory(p, A.t.options());
  const CUtensorMap ma = A.map(), mb = B.map();
  auto map_of = [&](const OutRows& o) { return o.tma && o.d != nullptr ? out_rows_map(o) : ma; };
  if constexpr (ACT == kActNone) {
    const typename BiasEpilogue<FP16>::Args args{map_of(r.out[0]), r.out[0], r.bias};
    launch_pair_gemm<KIND, BiasEpilogue<FP16>>(ma, mb, parts, args, p, device, stream);
  } else {
    typename ActGradEpilogue<FP16, ACT>::Args args;
    for (int h = 0; h < ActGradEpilogue<FP16, ACT>::H; ++h) {
      args.map_dx[h] = map_of(r.out[h]);
      args.dx[h] = r.out[h];
    }
    args.map_a = map_of(r.value);
    args.act = r.value;
    args.want_act = r.want_value;
    args.kept = r.kept;
    launch_pair_gemm<KIND, ActGradEpilogue<FP16, ACT>>(ma, mb, parts, args, p, device, stream);
  }
  if (p.split > 1)
    launch_overlapping(part_sum_kernel<FP16, ACT>, part_grid(p), dim3(kPartThreads), 0, stream, true,
                       PartSum{reinterpret_cast<const float*>(parts.data_ptr()), p, {r.out[0], r.out[1]}, r.bias, r.value,
                               r.want_value, r.kept});
}

void product(const Operand& A, const Operand& B, const Result& r, cudaStream_t stream) {
  const bool fp16 = A.t.scalar_type() == at::kHalf;
  const int device = A.t.get_device();
  auto typed = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (fp16) product_typed<true, ACT>(A, B, r, device, stream);
    else product_typed<false, ACT>(A, B, r, device, stream);
  };
  if (r.act == kActGelu) typed(std::integral_constant<int, kActGelu>{});
  else if (r.act == kActSwiglu) typed(std::integral_constant<int, kActSwiglu>{});
  else typed(std::integral_constant<int, kActNone>{});
}


// act(x') [R, F] of the codes.
at::Tensor decode(const Kept& kept, int64_t R, int64_t F, int64_t act, const at::TensorOptions& options, cudaStream_t stream) {
  const int64_t lda = (F + 15) / 16 * 16;
  at::Tensor a = at::empty({R, lda}, options).narrow(1, 0, F);
  if (act == kActNone) {
    int8_dequantize_launch(Int8Matrix{kept.data, nullptr, kept.exponents, R, F}, a, stream);
    return a;
  }
  const dim3 block = row_block((F + 3) / 4);
  const unsigned grid = (unsigned)((R + block.y - 1) / block.y);
  uint16_t* to = static_cast<uint16_t*>(a.data_ptr());
  if (options.dtype() == at::kHalf) {
    if (act == kActGelu) act_decode_kernel<true, kActGelu><<<grid, block, 0, stream>>>(kept, to, lda, (int)R, (int)F);
    else act_decode_kernel<true, kActSwiglu><<<grid, block, 0, stream>>>(kept, to, lda, (int)R, (int)F);
  } else {
    if (act == kActGelu) act_decode_kernel<false, kActGelu><<<grid, block, 0, stream>>>(kept, to, lda, (int)R, (int)F);
    else act_decode_kernel<false, kActSwiglu><<<grid, block, 0, stream>>>(kept, to, lda, (int)R, (int)F);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return a;
}

}  // namespace

void act8_check(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& bias, int64_t act) {
  const auto dt = x.scalar_type();
  DMAD_VALUE_CHECK(x.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf), "linear_act8: x must be bf16 or fp16 on CUDA");
  DMAD_VALUE_CHECK(w.dim() == 2 && w.scalar_type() == dt && w.device() == x.device(),
                   "linear_act8: w must be a matrix of x's type on its device, got " + std::string(dtype_name(w.scalar_type())) +
                       " " + shape_text(w));
  const int64_t F = w.size(1);
  DMAD_VALUE_CHECK(F >= 1 && F <= (1 << 23) && w.size(0) <= (1 << 24), "linear_act8: w " + shape_text(w) + ": sizes out of range");
  DMAD_VALUE_CHECK(x.dim() >= 1 && x.size(-1) == halves(act) * F,
                   "linear_act8: x " + shape_text(x) + " must have " + num(halves(act) * F) + " columns for w " + shape_text(w));
  checked_bias(bias, w.size(0), x.device(), "linear_act8");
}

// (y, codes, exponents) of x [..., H F], W [N, F] (checked); the codes [R H, ..] where `keep` is set.
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_forward(const at::Tensor& x, const at::Tensor& w,
                                                            const c10::optional<at::Tensor>& bias, int64_t act, bool keep) {
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t N = w.size(0), F = w.size(1), H = halves(act);
  const at::Tensor x2 = int8_rows(x, "linear_act8");
  const int64_t R = x2.size(0);
  DMAD_VALUE_CHECK(R * H <= INT32_MAX - 256, "linear_act8: too many rows");
  const auto plain = x.options().requires_grad(false);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const auto b = bias.has_value() && bias->defined() ? c10::optional<at::Tensor>(bias->contiguous()) : c10::nullopt;
  at::Tensor data, exponents;
  Kept kept{nullptr, nullptr};
  if (keep) {
    data = at::empty({R * H, int8_row_bytes(F)}, plain.dtype(at::kChar));
    exponents = at::empty({R * H, (F + kInt8Block - 1) / kInt8Block}, plain.dtype(at::kByte));
    kept = kept_of(data, exponents);
  }
  // copies before the pass over x, so that the product may overlap that pass without reading anything younger
  const bool some = R > 0 && N > 0;
  const at::Tensor wt = some ? tma_rows(w, stream) : w;
  at::Tensor a;
  bool copied = act != kActNone;
  if (act == kActNone) {
    if (some && !tma_readable(x2)) {
      a = encode(x2, F, act, kept, stream);  // a copy and the codes in one pass
      copied = true;
    } else {
      a = x2;
      if (keep) int8_quantize_launch(x2, Int8Matrix{kept.data, nullptr, kept.exponents, R, F}, stream);
    }
  } else {
    a = encode(x2, F, act, kept, stream);
  }
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, plain);
  if (some) {
    Result r;
    r.out[0] = out_rows(y.data_ptr(), N, R, N);
    r.bias = float_row(b);
    r.early = copied ? 1 : keep ? 2 : 0;
    r.b_old = true;
    product(Operand{a, false}, Operand{wt, false}, r, stream);
  }
  return {y, data, exponents};
}

// Gradients of x (shape [R, H F]), w and bias (undefined where they are not wanted).
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_backward(const at::Tensor& g, const at::Tensor& w, const at::Tensor& data,
                                                             const at::Tensor& exponents, int64_t act, int64_t R,
                                                             bool want_x, bool want_w, bool want_b, at::ScalarType bias_type) {
  c10::cuda::CUDAGuard guard(g.device());
  const int64_t N = w.size(0), F = w.size(1), H = halves(act);
  const auto plain = w.options().requires_grad(false);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor dx, dw, db;
  if (want_x) dx = at::empty({R, H * F}, plain);
  if (R == 0 || N == 0) {
    if (want_x) dx.zero_();
    if (want_w) dw = at::zeros({N, F}, plain);
    if (want_b) db = at::zeros({N}, plain.dtype(bias_type));
    return {dx, dw, db};
  }
  // Copies, then the passes that only read them and the codes, then the products, each overlapping the end of the kernel
  // before it: the first one reads nothing that those passes write (early 2) or, for want_w, what the one before did.
  const at::Tensor gt = tma_rows(g.dim() == 2 ? g : g.reshape({R, N}), stream);
  const at::Tensor wt = want_x ? tma_rows(w, stream) : w;
  const Kept kept = data.defined() ? kept_of(data, exponents) : Kept{nullptr, nullptr};
  at::Tensor a;  // act(x')
  if (want_b) db = column_sum(gt, bias_type, stream);
  if (want_w && (act == kActNone || !want_x)) a = decode(kept, R, F, act, plain, stream);
  if (want_x) {
    Result r;
    r.early = want_b || a.defined() ? 2 : 0;
    for (int h = 0; h < H; ++h) r.out[h] = out_rows(static_cast<uint16_t*>(dx.data_ptr()) + h * F, H * F, R, F);
    r.act = (int)act;
    r.kept = kept;
    if (act != kActNone && want_w) {
      a = at::empty({R, (F + 15) / 16 * 16}, plain);
      r.value = out_rows(a.data_ptr(), a.stride(0), R, a.size(1));  // columns past F may be written, nothing reads them
      a = a.narrow(1, 0, F);
      r.want_value = true;
    }
    product(Operand{gt, false}, Operand{wt, true}, r, stream);
  }
  if (want_w) {
    dw = at::empty({N, F}, plain);
    Result r;
    r.early = 1;
    r.out[0] = out_rows(dw.data_ptr(), F, N, F);
    product(Operand{gt, true}, Operand{a, true}, r, stream);
  }
  return {dx, dw, db};
}

}  // namespace dmad
