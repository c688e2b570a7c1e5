// Per-head RMSNorm of queries and keys with the position rotation in the same pass, and its backward.
//
//   n = x / sqrt(mean(x^2) + eps),   y = n * w,   out = Rot(y)              (per row and head of hd elements)
//   gy = Rot^-1(g),   dw = sum gy * n,   dx = (gy w - n mean(gy w n)) / sqrt(mean(x^2) + eps)
//
// Rot turns the first `rot` elements of a head: pairs (2i, 2i + 1) (interleaved) or (i, i + rot / 2) (halves) by the
// angle whose cosine and sine stand in row t, column i of the tables; t is the row's entry of `positions`, or
// r % T.  Everything is fp32 between the load and the one rounding at the store.
//
// Bound by HBM: the forward reads and writes q and k once, the backward reads g and x and writes dx; the
// statistics are taken again from x, which is in registers anyway, so nothing is kept between the passes.  A
// head is held by a group of G lanes, eight elements a lane (16-byte accesses of 16-bit types, streamed past the
// caches: nothing is read twice), and a group takes U heads of one row at a time: U loads in flight, one read of the
// row's angles.  gridDim.y separates q from k, so a thread has one weight slice and one gradient accumulator.  dw:
// per-thread sums over the tasks of a persistent grid, one partial row a block, and a second kernel that adds the
// partials in a fixed order.
// Measured at 37966 rows of 40 + 40 heads of 128, bf16, pairs: forward 255 us (6.1 TB/s), backward 404 us (5.8 TB/s; with
// U = 4 instead of 8 and cached accesses 497 us; with the next task's loads issued ahead, U = 2, 690 us).  Halves, whose
// partners come by shuffles: 300 and 459 us.  fp32, half as many rows: pairs 245 and 362 us, halves 262 and 364 us (the
// forward of these holds four heads of fp32 in 64 registers and spills 132 bytes).
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "checks.h"
#include "common.cuh"

namespace dmad {

int* device_status_ptr(int device);

namespace {

constexpr int kThreads = 256;

// How the angles are applied.  The vectorised forms need table rows of whole 16-byte pieces and, for halves,
// partners that are whole lanes apart; kAny takes every other size one element at a time.
enum RotMode { kNone = 0, kPairs = 1, kHalves = 2, kAny = 3 };

struct Side {  // the queries or the keys
  const void* x;
  const void* g;
  void* out;      // forward: the result; backward: dx
  int64_t xr, xh, gr, gh, orow, oh;  // row and head strides
  const void* w;  // nullptr: ones
  int wtype;      // 0 fp32, 1 bf16, 2 fp16
  int H, chunks;
  float* partial;  // backward: [gridDim.x, hd] sums of gy * n, or nullptr
};

struct Params {
  Side side[2];
  const float* cosT;
  const float* sinT;
  const void* positions;
  int pos64;
  int64_t T;
  int64_t R;
  int hd, rot, interleaved;
  float eps;
  int* status;
};

// Eight elements as they lie in memory: they stay packed until their head is worked on, which halves the registers
// that the loads in flight occupy.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          f[4 * i + j] = __uint_as_float(w[j]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          f[2 * j] = __uint_as_float(w[j] << 16);
          f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          f[2 * j] = h.x;
          f[2 * j + 1] = h.y;
        }
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        w[i] = f2_to_bf16x2(f[2 * i], f[2 * i + 1]);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}

__device__ __forceinline__ float load_any(const void* p, int type, int i) {
  if (type == 0) return static_cast<const float*>(p)[i];
  if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  else return __half2float(v);
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The angles that a lane needs of table row t.  kPairs: c[0..3] for its four pairs; kHalves: c[0..7] for its
// eight elements.  Elements past `rot` keep (1, 0).
template <int MODE>
struct Angles {
  float c[MODE == kPairs ? 4 : 8], s[MODE == kPairs ? 4 : 8];
  int64_t off;  // kAny: offset of the row, -1 if there is none

  __device__ __forceinline__ void load(const Params& p, int64_t row, int e0, bool valid) {
    if constexpr (MODE == kNone) return;
    constexpr int N = MODE == kPairs ? 4 : 8;
    int64_t t = 0;
    if (valid) {
      t = p.positions == nullptr ? (row < p.T ? row : row % p.T)
          : p.pos64              ? static_cast<const int64_t*>(p.positions)[row]
                                 : static_cast<const int*>(p.positions)[row];
    }
    const bool bad = t < 0 || t >= p.T;
    if (bad) atomicCAS(p.status, 0, 6);  // bounds: the rotated elements become NaN
    const int half = p.rot >> 1;
    if constexpr (MODE == kAny) {
      off = bad ? -1 : t * half;
    } else {
      const int col = MODE == kPairs ? e0 >> 1 : (e0 < half ? e0 : e0 - half);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        c[i] = bad ? __int_as_float(0x7fffffff) : 1.f;
        s[i] = bad ? __int_as_float(0x7fffffff) : 0.f;
      }
      if (e0 < p.rot && !bad) {
        const float4* pc = reinterpret_cast<const float4*>(p.cosT + t * half + col);
        const float4* ps = reinterpret_cast<const float4*>(p.sinT + t * half + col);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
          const float4 a = __ldg(pc + i), b = __ldg(ps + i);
          c[4 * i] = a.x; c[4 * i + 1] = a.y; c[4 * i + 2] = a.z; c[4 * i + 3] = a.w;
          s[4 * i] = b.x; s[4 * i + 1] = b.y; s[4 * i + 2] = b.z; s[4 * i + 3] = b.w;
        }
      }
    }
  }

  // y <- the rotated y (forward) or the back-rotated y (INV).  other(i): element i of the head, for kAny.
  template <bool INV, typename F>
  __device__ __forceinline__ void apply(const Params& p, int e0, float (&y)[8], F other) const {
    if constexpr (MODE == kPairs) {
      if (e0 >= p.rot) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = y[2 * j], b = y[2 * j + 1], sn = INV ? -s[j] : s[j];
        y[2 * j] = a * c[j] - b * sn;
        y[2 * j + 1] = b * c[j] + a * sn;
      }
    } else if constexpr (MODE == kHalves) {
      const int half = p.rot >> 1;
      const int from = e0 < half ? half >> 3 : e0 < p.rot ? -(half >> 3) : 0;
      const float sign = (e0 < half) == INV ? 1.f : -1.f;  // first half: a c - b s; second half: b c + a s
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float o = __shfl_sync(0xffffffffu, y[j], lane + from);
        if (e0 < p.rot) y[j] = y[j] * c[j] + sign * s[j] * o;
      }
    } else if constexpr (MODE == kAny) {
      const int half = p.rot >> 1;
      float z[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = e0 + j;
        z[j] = y[j];
        if (i < p.rot) {
          const bool first = p.interleaved ? (j & 1) == 0 : i < half;
          const int col = p.interleaved ? i >> 1 : first ? i : i - half;
          const float o = p.interleaved ? y[j ^ 1] : other(first ? i + half : i - half);
          const float cc = off < 0 ? __int_as_float(0x7fffffff) : __ldg(p.cosT + off + col);
          const float ss = off < 0 ? __int_as_float(0x7fffffff) : __ldg(p.sinT + off + col);
          z[j] = y[j] * cc + (first == INV ? ss : -ss) * o;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = z[j];
    }
  }
};

__device__ __forceinline__ void split_task(int64_t task, int64_t tasks, int chunks, int64_t& row, int& chunk) {
  if (tasks <= 0x7fffffff) {
    row = (uint32_t)task / (uint32_t)chunks;
    chunk = (int)((uint32_t)task - (uint32_t)row * (uint32_t)chunks);
  } else {
    row = task / chunks;
    chunk = (int)(task - row * chunks);
  }
}

template <typename T, int G, int MODE, int U>
__global__ void __launch_bounds__(kThreads, 4) head_norm_fwd_kernel(const __grid_constant__ Params p) {
  const Side& sd = p.side[blockIdx.y];
  const int lane = threadIdx.x & (G - 1), e0 = lane * 8;
  const bool in = e0 < p.hd;
  const int64_t tasks = p.R * sd.chunks;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / G);
  float w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = in && sd.w != nullptr ? load_any(sd.w, sd.wtype, e0 + j) : 1.f;
  const float inv_hd = 1.f / (float)p.hd;
  const int group = threadIdx.x / G;
  // all lanes of a warp stay in the loop together: the sums below are warp-wide shuffles
  for (int64_t first = (int64_t)blockIdx.x * (kThreads / G) + (group & ~(32 / G - 1)); first < tasks; first += stride) {
    const int64_t task = first + (group & (32 / G - 1));
    const bool valid = task < tasks;
    int64_t row = 0;
    int chunk = 0;
    if (valid) split_task(task, tasks, sd.chunks, row, chunk);
    const T* x = static_cast<const T*>(sd.x) + row * sd.xr + (int64_t)chunk * U * sd.xh;
    T* o = static_cast<T*>(sd.out) + row * sd.orow + (int64_t)chunk * U * sd.oh;
    const int nh = valid ? min(U, sd.H - chunk * U) : 0;
    Raw8<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (in && u < nh) raw[u].load(x + u * sd.xh + e0);
      else raw[u].zero();
    }
    Angles<MODE> ang;
    ang.load(p, row, e0, valid);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      raw[u].unpack(f);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
      const float r = rsqrtf(group_sum<G>(ss) * inv_hd + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
      ang.template apply<false>(p, e0, f, [&](int i) {
        return u < nh ? to_float(x[u * sd.xh + i]) * r * (sd.w != nullptr ? load_any(sd.w, sd.wtype, i) : 1.f) : 0.f;
      });
      if (in && u < nh) store8(o + u * sd.oh + e0, f);
    }
  }
}

template <typename T, int G, int MODE, int U>
__global__ void __launch_bounds__(kThreads, 2) head_norm_bwd_kernel(const __grid_constant__ Params p) {
  __shared__ float red[kThreads * 8];
  const Side& sd = p.side[blockIdx.y];
  const int lane = threadIdx.x & (G - 1), e0 = lane * 8;
  const bool in = e0 < p.hd;
  const int64_t tasks = p.R * sd.chunks;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / G);
  float w[8], acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = in && sd.w != nullptr ? load_any(sd.w, sd.wtype, e0 + j) : 1.f;
    acc[j] = 0.f;
  }
  const float inv_hd = 1.f / (float)p.hd;
  const int group = threadIdx.x / G;
  for (int64_t first = (int64_t)blockIdx.x * (kThreads / G) + (group & ~(32 / G - 1)); first < tasks; first += stride) {
    const int64_t task = first + (group & (32 / G - 1));
    const bool valid = task < tasks;
    int64_t row = 0;
    int chunk = 0;
    if (valid) split_task(task, tasks, sd.chunks, row, chunk);
    const T* x = static_cast<const T*>(sd.x) + row * sd.xr + (int64_t)chunk * U * sd.xh;
    const T* g = static_cast<const T*>(sd.g) + row * sd.gr + (int64_t)chunk * U * sd.gh;
    T* o = static_cast<T*>(sd.out) + row * sd.orow + (int64_t)chunk * U * sd.oh;
    const int nh = valid ? min(U, sd.H - chunk * U) : 0;
    Raw8<T> rawx[U], rawg[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (in && u < nh) {
        rawx[u].load(x + u * sd.xh + e0);
        rawg[u].load(g + u * sd.gh + e0);
      } else {
        rawx[u].zero();
        rawg[u].zero();
      }
    }
    Angles<MODE> ang;
    ang.load(p, row, e0, valid);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8], d[8];
      rawx[u].unpack(f);
      rawg[u].unpack(d);
      ang.template apply<true>(p, e0, d, [&](int i) { return u < nh ? to_float(g[u * sd.gh + i]) : 0.f; });
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fmaf(f[j], f[j], ss);
        dot = fmaf(d[j] * w[j], f[j], dot);
      }
      const float r = rsqrtf(group_sum<G>(ss) * inv_hd + p.eps);
      const float c = group_sum<G>(dot) * r * inv_hd;  // mean(gy w n)
      float dx[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = f[j] * r;
        if (u < nh) acc[j] = fmaf(d[j], n, acc[j]);
        dx[j] = (d[j] * w[j] - n * c) * r;
      }
      if (in && u < nh) store8(o + u * sd.oh + e0, dx);
    }
  }
  if (sd.partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[threadIdx.x * 8 + j] = acc[j];
  __syncthreads();
  // red[group][lane * 8 + j]: add the block's groups in order
  for (int i = threadIdx.x; i < p.hd; i += kThreads) {
    float t = 0.f;
    for (int q = 0; q < kThreads / G; ++q) t += red[q * G * 8 + i];
    sd.partial[(int64_t)blockIdx.x * p.hd + i] = t;
  }
}

// dw[i] = sum over the blocks of partial[block][i], in a fixed order.
__global__ void __launch_bounds__(1024)
head_norm_dw_kernel(const float* __restrict__ pq, const float* __restrict__ pk, int blocks, int hd, void* dwq, int tq,
                    void* dwk, int tk) {
  __shared__ float red[32][33];
  const float* part = blockIdx.y == 0 ? pq : pk;
  void* dw = blockIdx.y == 0 ? dwq : dwk;
  const int type = blockIdx.y == 0 ? tq : tk;
  if (dw == nullptr) return;
  const int i = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (i < hd)
    for (int b = threadIdx.y; b < blocks; b += 32) t += part[(int64_t)b * hd + i];
  red[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && i < hd) {
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < 32; ++b) sum += red[b][threadIdx.x];
    if (type == 0) static_cast<float*>(dw)[i] = sum;
    else if (type == 1) static_cast<__nv_bfloat16*>(dw)[i] = __float2bfloat16_rn(sum);
    else static_cast<__half*>(dw)[i] = __float2half_rn(sum);
  }
}

int float_type(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }

const char* const kOp = "qk_head_norm_rope: ";

bool rows_ok(const at::Tensor& t) {
  const int64_t per16 = 16 / (int64_t)t.element_size();
  return t.numel() == 0 || (t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) % per16 == 0) &&
                            (t.size(0) == 1 || t.stride(0) % per16 == 0) &&
                            reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0);
}

// A [R, H, hd] operand that the kernels can read: the tensor itself or a contiguous copy.
at::Tensor readable(const at::Tensor& t) { return rows_ok(t) ? t : t.contiguous(); }

void check_heads(const at::Tensor& t, const at::Tensor& q, int64_t H, const char* name, bool in_place) {
  DMAD_VALUE_CHECK(t.device() == q.device() && t.scalar_type() == q.scalar_type() && t.dim() == 3 &&
                       t.size(0) == q.size(0) && t.size(1) == H && t.size(2) == q.size(2),
                   std::string(kOp) + name + " must be (" + num(q.size(0)) + ", " + num(H) + ", " + num(q.size(2)) +
                       ") of the type and on the device of q, got " + shape_text(t));
  DMAD_VALUE_CHECK(!in_place || rows_ok(t), std::string(kOp) + name +
                                                ": heads must be contiguous, strides and the start multiples of 16 bytes");
}

struct Prepared {  // what the kernels' parameters point into
  at::Tensor x[2], w[2], cosT, sinT, positions;
  RotMode mode = kNone;
};

Prepared fill_common(Params& p, const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& wq,
                     const c10::optional<at::Tensor>& wk, const c10::optional<at::Tensor>& cosT,
                     const c10::optional<at::Tensor>& sinT, const c10::optional<at::Tensor>& positions, double eps,
                     bool interleaved) {
  Prepared keep;
  const std::string op(kOp);
  DMAD_VALUE_CHECK(q.dim() == 3 && k.dim() == 3 && is_float_type(q.scalar_type()),
                   op + "q and k must be [R, heads, hd] in bf16, fp16 or fp32, got " + shape_text(q) + " and " + shape_text(k));
  const int64_t R = q.size(0), hd = q.size(2);
  DMAD_VALUE_CHECK(hd >= 8 && hd <= 256 && hd % 8 == 0 && q.size(1) >= 1 && k.size(1) >= 1 && q.size(1) <= 65536 &&
                       k.size(1) <= 65536,
                   op + "the head size must be a multiple of 8 up to 256 and q and k have heads, got " + shape_text(q) +
                       " and " + shape_text(k));
  check_heads(k, q, k.size(1), "k", false);
  DMAD_VALUE_CHECK(q.is_cuda(), op + "the native kernel takes CUDA tensors");
  const at::Tensor* xs[2] = {&q, &k};
  const c10::optional<at::Tensor>* ws[2] = {&wq, &wk};
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    keep.x[i] = readable(*xs[i]);
    s.x = keep.x[i].data_ptr();
    s.xr = keep.x[i].stride(0);
    s.xh = keep.x[i].stride(1);
    s.H = (int)xs[i]->size(1);
    s.g = nullptr;
    s.gr = s.gh = 0;
    s.partial = nullptr;
    s.w = nullptr;
    s.wtype = 0;
    if (ws[i]->has_value() && (*ws[i])->defined()) {
      const at::Tensor& w = **ws[i];
      DMAD_VALUE_CHECK(w.device() == q.device() && w.dim() == 1 && w.size(0) == hd && is_float_type(w.scalar_type()),
                       op + (i ? "wk" : "wq") + " must be bf16, fp16 or fp32 (" + num(hd) + ",) on the device of q, got " +
                           dtype_name(w.scalar_type()) + " " + shape_text(w));
      keep.w[i] = w.contiguous();
      s.w = keep.w[i].data_ptr();
      s.wtype = float_type(w);
    }
  }
  p.R = R;
  p.hd = (int)hd;
  p.rot = 0;
  p.T = 1;
  p.cosT = p.sinT = nullptr;
  p.positions = nullptr;
  p.pos64 = 0;
  p.interleaved = interleaved ? 1 : 0;
  p.eps = (float)eps;
  p.status = device_status_ptr(q.get_device());
  const bool has_cos = cosT.has_value() && cosT->defined(), has_sin = sinT.has_value() && sinT->defined();
  const bool has_pos = positions.has_value() && positions->defined();
  DMAD_VALUE_CHECK(has_cos == has_sin && (has_cos || !has_pos), op + "cos and sin come together, and positions with them");
  if (!has_cos) return keep;
  DMAD_VALUE_CHECK(cosT->dim() == 2 && cosT->sizes() == sinT->sizes() && cosT->size(0) >= 1 && 2 * cosT->size(1) <= hd,
                   op + "cos and sin must be [T, rot / 2] with T >= 1 and rot <= " + num(hd) + ", got " +
                       shape_text(*cosT) + " and " + shape_text(*sinT));
  DMAD_VALUE_CHECK(cosT->device() == q.device() && sinT->device() == q.device() && at::isFloatingType(cosT->scalar_type()) &&
                       at::isFloatingType(sinT->scalar_type()) && !cosT->requires_grad() && !sinT->requires_grad(),
                   op + "cos and sin are constant floating-point tables on the device of q (no gradient)");
  keep.cosT = cosT->to(at::kFloat).contiguous();
  keep.sinT = sinT->to(at::kFloat).contiguous();
  if (has_pos) {
    DMAD_VALUE_CHECK(positions->device() == q.device() && positions->dim() == 1 && positions->size(0) == R &&
                         (positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt),
                     op + "positions must be int32 or int64 (" + num(R) + ",) on the device of q, got " +
                         shape_text(*positions));
  }
  p.rot = (int)cosT->size(1) * 2;
  if (p.rot == 0) return keep;
  p.T = cosT->size(0);
  p.cosT = keep.cosT.data_ptr<float>();
  p.sinT = keep.sinT.data_ptr<float>();
  if (has_pos) {
    keep.positions = positions->contiguous();
    p.positions = keep.positions.data_ptr();
    p.pos64 = positions->scalar_type() == at::kLong ? 1 : 0;
  }
  const bool tables16 = reinterpret_cast<uintptr_t>(p.cosT) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sinT) % 16 == 0;
  if (interleaved) keep.mode = tables16 && p.rot % 8 == 0 ? kPairs : kAny;
  else keep.mode = tables16 && p.rot % 16 == 0 ? kHalves : kAny;
  return keep;
}

template <typename F>
void dispatch_mode(RotMode m, F f) {
  if (m == kNone) f(std::integral_constant<int, kNone>{});
  else if (m == kPairs) f(std::integral_constant<int, kPairs>{});
  else if (m == kHalves) f(std::integral_constant<int, kHalves>{});
  else f(std::integral_constant<int, kAny>{});
}
template <typename F>
void dispatch_group(int hd, F f) {
  if (hd <= 32) f(std::integral_constant<int, 4>{});
  else if (hd <= 64) f(std::integral_constant<int, 8>{});
  else if (hd <= 128) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}
template <typename F>
void dispatch_type(at::ScalarType t, F f) {
  if (t == at::kBFloat16) f(__nv_bfloat16{});
  else if (t == at::kHalf) f(__half{});
  else f(float{});
}

int64_t blocks_for(const Params& p, int G, int64_t most) {
  const int per = kThreads / G;
  int64_t b = 1;
  for (const Side& s : p.side) b = std::max(b, (p.R * s.chunks + per - 1) / per);
  return std::min(b, most);
}

}  // namespace

// Rot(norm(q) * wq), Rot(norm(k) * wk) per head, contiguous.
std::tuple<at::Tensor, at::Tensor> head_norm_rope_fwd(const at::Tensor& q, const at::Tensor& k,
                                                      c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk,
                                                      c10::optional<at::Tensor> cosT, c10::optional<at::Tensor> sinT,
                                                      c10::optional<at::Tensor> positions, double eps,
                                                      bool interleaved) {
  c10::cuda::OptionalCUDAGuard guard;
  if (q.is_cuda()) guard.set_device(q.device());
  Params p;
  const Prepared keep = fill_common(p, q, k, wq, wk, cosT, sinT, positions, eps, interleaved);
  const auto plain = q.options().requires_grad(false);
  at::Tensor outs[2] = {at::empty(q.sizes(), plain), at::empty(k.sizes(), plain)};
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    s.orow = outs[i].stride(0);
    s.oh = outs[i].stride(1);
    s.out = outs[i].data_ptr();
  }
  if (p.R == 0) return {outs[0], outs[1]};
  const RotMode mode = keep.mode;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int sms = sm_count(q.get_device());
  dispatch_type(q.scalar_type(), [&](auto tag) {
    using T = decltype(tag);
    dispatch_group(p.hd, [&](auto g) {
      dispatch_mode(mode, [&](auto m) {
        constexpr int U = 4;
        for (Side& s : p.side) s.chunks = (s.H + U - 1) / U;
        const dim3 grid((unsigned)blocks_for(p, g, (int64_t)sms * 16), 2);
        head_norm_fwd_kernel<T, decltype(g)::value, decltype(m)::value, U><<<grid, kThreads, 0, stream>>>(p);
      });
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {outs[0], outs[1]};
}

// dq, dk of the forward given gq, gk (gradients of its results) and its inputs; dwq, dwk [hd] where wanted.
void head_norm_rope_bwd(const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k,
                        c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk, c10::optional<at::Tensor> cosT,
                        c10::optional<at::Tensor> sinT, c10::optional<at::Tensor> positions, at::Tensor& dq,
                        at::Tensor& dk, c10::optional<at::Tensor> dwq, c10::optional<at::Tensor> dwk, double eps,
                        bool interleaved) {
  c10::cuda::OptionalCUDAGuard guard;
  if (q.is_cuda()) guard.set_device(q.device());
  Params p;
  const Prepared keep = fill_common(p, q, k, wq, wk, cosT, sinT, positions, eps, interleaved);
  const RotMode mode = keep.mode;
  const at::Tensor* gs[2] = {&gq, &gk};
  at::Tensor* outs[2] = {&dq, &dk};
  const c10::optional<at::Tensor>* dws[2] = {&dwq, &dwk};
  at::Tensor g[2];
  void* dwp[2] = {nullptr, nullptr};
  int dwt[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    check_heads(*gs[i], q, s.H, i ? "gk" : "gq", false);
    check_heads(*outs[i], q, s.H, i ? "dk" : "dq", true);
    g[i] = readable(*gs[i]);
    s.g = g[i].data_ptr();
    s.gr = g[i].stride(0);
    s.gh = g[i].stride(1);
    s.out = outs[i]->data_ptr();
    s.orow = outs[i]->stride(0);
    s.oh = outs[i]->stride(1);
    if (dws[i]->has_value() && (*dws[i])->defined()) {
      const at::Tensor& dw = **dws[i];
      DMAD_VALUE_CHECK(dw.device() == q.device() && dw.dim() == 1 && dw.size(0) == p.hd && dw.is_contiguous() &&
                           is_float_type(dw.scalar_type()),
                       std::string(kOp) + "a weight gradient must be contiguous bf16, fp16 or fp32 (" + num(p.hd) + ",)");
      dwp[i] = dw.data_ptr();
      dwt[i] = float_type(dw);
    }
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int sms = sm_count(q.get_device());
  const bool want_dw = dwp[0] != nullptr || dwp[1] != nullptr;
  at::Tensor partial;
  int blocks = 0;
  if (p.R > 0) {
    dispatch_type(q.scalar_type(), [&](auto tag) {
      using T = decltype(tag);
      dispatch_group(p.hd, [&](auto g) {
        dispatch_mode(mode, [&](auto m) {
          constexpr int U = sizeof(T) == 4 ? 4 : 8;
          for (Side& s : p.side) s.chunks = (s.H + U - 1) / U;
          blocks = (int)blocks_for(p, g, (int64_t)sms * 2);
          if (want_dw) {
            partial = at::empty({2, blocks, p.hd}, q.options().dtype(at::kFloat));
            for (int i = 0; i < 2; ++i)
              p.side[i].partial = dwp[i] != nullptr ? partial.data_ptr<float>() + (int64_t)i * blocks * p.hd : nullptr;
          }
          head_norm_bwd_kernel<T, decltype(g)::value, decltype(m)::value, U>
              <<<dim3((unsigned)blocks, 2), kThreads, 0, stream>>>(p);
        });
      });
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (want_dw) {
    head_norm_dw_kernel<<<dim3((p.hd + 31) / 32, 2), dim3(32, 32), 0, stream>>>(p.side[0].partial, p.side[1].partial,
                                                                              blocks, p.hd, dwp[0], dwt[0], dwp[1], dwt[1]);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace dmad
