// tcgen05 GEMMs of 8-bit integers for sm_100a.
//
//   D[M, N] = ra[m] rb[n] * sum_k A[m, k] B[n, k] + bias[n]          (bf16 or fp16 out)
//
// A and B are codes of -127 .. 127 with a scale a row (int8.cuh), multiplied on the tensor core (kind::i8) with exact int32
// sums (K <= 133144: 2^31 / 127^2), so the only roundings are the epilogue's: the factors, the bias, and one to the result's
// type.  Three kernels, by the rows of A: for one, dot products that stream the weight; up to kSmallBN, MMAs whose rows are the
// weight's; above that, pairs of CTAs on 256 x 256 tiles (gemm_pair.cuh).
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.cuh"
#include "gemm_pair.cuh"
#include "int8_host.h"
#include "row_factors.cuh"

namespace dmad {
namespace {

constexpr int64_t kMaxK = 133144;
constexpr int kBM = 128;            // weight rows of a tile of the few-rows kernel
constexpr int kBK = 128;            // columns of K of a stage
constexpr int kABytes = kBM * 128;  // 16 KB

struct Factors {
  const float* ra;
  const float* rb;
  FloatRow bias;
};

// ---------------------------------------------------------------- CTA pairs
// Factors and bias on the accumulators of gemm_pair.cuh.  Bound by the tensor core (92 % busy at 8192 x 8192 x 8192): 3.2
// POP/s there, 37966 x 30720 x 5120 3.9 to 4.2 ms in short runs and 4.4 to 5.1 ms over seconds, by the card and the clock that
// the power limit leaves.  N = 30719, whose rows of 16-bit results start off 16 bytes, 8 % more (4.48 against 4.16 ms).
template <bool FP16>
struct ScaleEpilogue {
  static constexpr int kStages = 6, kWarps = 8, kOutBytes = 2048;
  static constexpr bool kShared = true, kAhead = true;
  struct Args {
    CUtensorMap map;
    OutRows out;
    Factors f;
  };
  const Args& a;
  const PairGemm& p;
  const EpiPlace at;
  int m0, n0, m0_next, n0_next;
  float ra, ra_next;
  float2 cf;
  bool far;
  const float2* col;

  __device__ __forceinline__ ScaleEpilogue(const Args& a, const PairGemm& p, const EpiPlace& at) : a(a), p(p), at(at) {}
  __device__ __forceinline__ void fetch(int item) {
    int tm, tn;
    p.tile(item, tm, tn);
    m0_next = tm * kPairM + (int)at.rank * kPairHalf + at.wq * 32;
    n0_next = tn * kPairN;
    const int n = min(n0_next + at.thread, p.N - 1);
    cf = make_float2(__ldg(a.f.rb + n), a.f.bias.at(n));
    ra_next = m0_next + at.lane < p.M ? __ldg(a.f.ra + m0_next + at.lane) : 1.f;
  }
  __device__ __forceinline__ void first(int item) { fetch(item); }
  __device__ __forceinline__ void begin(int, int, int parity) {
    // (the buffer's last readers are two tiles back, behind the barrier between)
    col = at.col + parity * kPairN;
    at.col[parity * kPairN + at.thread] = cf;
    m0 = m0_next;
    n0 = n0_next;
    ra = ra_next;
    far = __any_sync(0xffffffffu, far_out(ra));
  }
  __device__ __forceinline__ void met(int next) {  // the next tile's factors are read while this one is stored
    if (next >= 0) fetch(next);
  }
  __device__ __forceinline__ void chunk(int c, const uint32_t (&v)[32]) {
    const int nc = n0 + c * 32;
    if (nc >= p.N || m0 >= p.M) return;
    uint32_t o[16];
    const float4* f4 = reinterpret_cast<const float4*>(col + c * 32);
    if (far) {  // one vote a tile, so that the warp stays together
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const float4 f = f4[q];
        const float x = __int2float_rn((int)v[2 * q]), y = __int2float_rn((int)v[2 * q + 1]);
        const bool out = far_out(ra);
        o[q] = pack16<FP16>(out ? apply_factors_far(x, ra, f.x, f.y) : apply_factors(x, ra, f.x, f.y),
                            out ? apply_factors_far(y, ra, f.z, f.w) : apply_factors(y, ra, f.z, f.w));
      }
    } else {
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const float4 f = f4[q];
        o[q] = pack16<FP16>(apply_factors(__int2float_rn((int)v[2 * q]), ra, f.x, f.y),
                            apply_factors(__int2float_rn((int)v[2 * q + 1]), ra, f.z, f.w));
      }
    }
    if (at.lane == 0) tma_store_wait_read();
    __syncwarp();
    store_rows(a.out, &a.map, at.stage, m0, nc, o);
  }
};

// Sum of a tile's int32 parts (exact, whatever the order), factors, bias and the result's type: four columns a thread.
struct PartSum {
  const int* parts;
  PairGemm g;
  OutRows out;
  Factors f;
};

template <bool FP16>
__global__ void __launch_bounds__(kPartThreads) int8_part_sum_kernel(const __grid_constant__ PartSum p) {
  wait_for_previous_grid();
  int m, n;
  int64_t at;
  if (!part_place(p.g, m, n, at)) return;
  int4 sum = make_int4(0, 0, 0, 0);
  for (int s = 0; s < p.g.split; ++s) {
    const int4 v = *reinterpret_cast<const int4*>(p.parts + at + s * kPartStep);
    sum.x += v.x;
    sum.y += v.y;
    sum.z += v.z;
    sum.w += v.w;
  }
  const float ra = __ldg(p.f.ra + m);
  const bool far = far_out(ra);
  const int acc[4] = {sum.x, sum.y, sum.z, sum.w};
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(n + i, p.g.N - 1);
    const float x = __int2float_rn(acc[i]), rb = __ldg(p.f.rb + c), b = p.f.bias.at(c);
    y[i] = far ? apply_factors_far(x, ra, rb, b) : apply_factors(x, ra, rb, b);
  }
  store4<FP16>(p.out, m, n, y);
}

// ---------------------------------------------------------------- one row
// The weight's bytes are all there is.  A block takes a run of the weight's rows, its warps equal shares of the run's 512-byte
// pieces, eight loads in flight each all the time (across rows), and multiplies them with the codes of x by four-way dot
// products; no matrix instruction has to be fed, no second grid waits.  A row that two warps share is added up in shared
// memory (whole numbers: the same in any order).  x is coded by every block for itself, from registers into shared memory (a
// few KB from the L2), while the first loads of the weight are on their way.
// 15360 x 5120: 15.8 to 17.7 us with the weight in the L2, 17.6 us without (two rows, on the few-rows kernel behind a
// quantiser: 15.4 and 18.8), some 6 us of it launch, coding and the last loads: 30720 rows take 11.9 us more (6.6 TB/s).  1536 x
// 1536 3.7 us (two rows: 7.0).  Sixteen loads in flight: 18.8 us; four blocks of 64 registers an SM, which spill: 24.3.
constexpr int kVectorThreads = 256, kVectorDepth = 8;
constexpr int kVectorUnits = 4;                                            // units of 16 columns of x a thread
constexpr int kVectorMaxK = kVectorThreads * kVectorUnits * 16;            // 16384
constexpr int kVectorBlocks = 2;                                           // of an SM
constexpr int kVectorMaxRows = 8192;                                       // of a block: 32 KB of sums
constexpr int kVectorSmem = kVectorMaxK + 512 + 4 * kVectorMaxRows;

struct VectorParams {
  const void* x;    // 16 bits, or codes
  const int8_t* w;
  void* d;
  Factors f;        // ra: of codes
  int out_fp16;
  int N, K;
};

// T: the type of x, int8_t where it is coded.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kVectorThreads, kVectorBlocks) int8_vector_kernel(const VectorParams p) {
  extern __shared__ __align__(16) int8_t codes[];  // whole pieces of 512 columns, then the sums of the block's rows
  __shared__ uint32_t red[kVectorThreads / 32];
  constexpr int kWarps = kVectorThreads / 32;
  const int warp = warp_id(), lane = lane_id();
  const int row_bytes = (int)int8_row_bytes(p.K), pieces = (row_bytes + 511) / 512, tail = row_bytes - (pieces - 1) * 512;
  int* sums = reinterpret_cast<int*>(codes + pieces * 512);
  // rows n0 .. n0 + rows - 1 of the block, and pieces begin .. end - 1 of them of the warp
  const int n0 = (int)((int64_t)p.N * blockIdx.x / gridDim.x), rows = (int)((int64_t)p.N * (blockIdx.x + 1) / gridDim.x) - n0;
  const int total = rows * pieces;
  const int begin = (int)((int64_t)total * warp / kWarps), end = (int)((int64_t)total * (warp + 1) / kWarps);
  const int first_row = begin / pieces, first_piece = begin % pieces;
  // rows lie one behind the other: the next piece is 512 bytes on, or `tail` at a row's end
  const int8_t* at = p.w + (int64_t)(n0 + first_row) * row_bytes + first_piece * 512 + lane * 16;
  int to_load = end - begin, lp = pieces - 1 - first_piece;  // loads left; pieces of the row behind the next one
  const bool in_tail = lane * 16 < tail;
  uint4 w[kVectorDepth];
  auto load = [&](uint4& to) {
    to = make_uint4(0u, 0u, 0u, 0u);
    if (to_load > 0 && (lp > 0 || in_tail)) to = ld_stream(at);
    --to_load;
    at += lp > 0 ? 512 : tail;
    lp = lp > 0 ? lp - 1 : pieces - 1;
  };
#pragma unroll
  for (int i = 0; i < kVectorDepth; ++i) load(w[i]);

  for (int r = threadIdx.x; r < rows; r += kVectorThreads) sums[r] = 0;
  float ra;
  if constexpr (std::is_same_v<T, int8_t>) {
    for (int c = threadIdx.x * 16; c < pieces * 512; c += kVectorThreads * 16) {
      uint32_t q[4] = {0u, 0u, 0u, 0u};
      if (c < row_bytes) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const int8_t*>(p.x) + c));
        q[0] = v.x, q[1] = v.y, q[2] = v.z, q[3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // zeros past the columns, whatever is stored there
        const int left = p.K - c - 4 * i;
        if (left < 4) q[i] = left <= 0 ? 0u : q[i] & ((1u << (8 * left)) - 1u);
      }
      *reinterpret_cast<uint4*>(codes + c) = make_uint4(q[0], q[1], q[2], q[3]);
    }
    ra = __ldg(p.f.ra);
  } else {
    const T* x = static_cast<const T*>(p.x);
    Unit<T> u[kVectorUnits];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVectorUnits; ++i) {
      const int unit = threadIdx.x + i * kVectorThreads;
      if constexpr (ALIGNED) u[i] = load_unit<T, true>(x, unit * 16, p.K);
      else u[i] = load_unit_anywhere<T>(x, unit * 16, p.K);
      top = max(top, absmax_bits(u[i]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < kWarps ? red[lane] : 0u);
    float inv;
    ra = int8_row_scale(top, inv);
#pragma unroll
    for (int i = 0; i < kVectorUnits; ++i) {
      const int col = (int)(threadIdx.x + i * kVectorThreads) * 16;
      if (col >= pieces * 512) break;  // (units past the columns are zeros)
      uint32_t q[4] = {0u, 0u, 0u, 0u};
      if (top < kInfBits) int8_encode_row(u[i], ra, inv, q);
      *reinterpret_cast<uint4*>(codes + col) = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
  __syncthreads();

  int acc = 0, left = end - begin, cp = pieces - 1 - first_piece, row = first_row;  // pieces left; of the row behind this one
  const int8_t *x0 = codes + lane * 16, *xc = x0 + first_piece * 512;
  while (left > 0) {
#pragma unroll
    for (int i = 0; i < kVectorDepth; ++i) {
      const uint4 v = w[i];  // (zeros past the end)
      load(w[i]);
      const uint4 x = *reinterpret_cast<const uint4*>(xc);
      acc = __dp4a((int)v.x, (int)x.x, __dp4a((int)v.y, (int)x.y, __dp4a((int)v.z, (int)x.z, __dp4a((int)v.w, (int)x.w, acc))));
      xc += 512;
      --left;
      if (cp == 0 || left == 0) {  // the same for the whole warp
        const int sum = __reduce_add_sync(0xffffffffu, acc);
        if (lane == 0) atomicAdd(&sums[row], sum);
        acc = 0;
        if (left == 0) break;
        ++row;
        cp = pieces;
        xc = x0;
      }
      --cp;
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += kVectorThreads) {
    const int n = n0 + r;
    const float s = __int2float_rn(sums[r]), rb = __ldg(p.f.rb + n), b = p.f.bias.at(n);
    const float y = far_out(ra) ? apply_factors_far(s, ra, rb, b) : apply_factors(s, ra, rb, b);
    static_cast<uint16_t*>(p.d)[n] = (uint16_t)(p.out_fp16 ? pack16<true>(y, 0.f) : pack16<false>(y, 0.f));
  }
}

// ---------------------------------------------------------------- few rows
// For few rows of x, D^T = B A^T: 128 rows of the weight B are the MMA's 128 rows and x's rows its N, so up to 32
// tokens cost a tile of 32 columns, and the K loop of a tile is split over a cluster of up to six CTAs.  Each leaves its
// int32 part in its shared memory, [row of x][128 rows], and adds a share of the columns over all parts (exactly,
// whatever the order), applies factors and bias and stores runs of the output row.
//   warp 0      producer (a ring of as many stages as fit); with `early` the grid was launched to overlap the quantiser of
//               x: the weight's part of the first stages is loaded before waiting for it
//   warp 1      TMEM owner and MMAs
//   warps 2..5  accumulator to shared memory; all warps add and store
// Two CTAs fit an SM.  2 to 16 rows, 15360 x 5120: 15.4 to 16.4 us with the quantiser, the weight in the L2 (18.8 to 19.3 us
// without), bound by the weight's bytes and the two kernels' latency; 128 x 5120 x 15360 24.5 us (26.8).
constexpr int kSmallThreads = 192, kSmallStages = 5;
constexpr int kSmallBN = 128;

struct SmallBars {
  float2 col[kBM];  // factor and bias of the tile's weight rows
  uint64_t full[kSmallStages], empty[kSmallStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct SmallParams {
  void* d;
  int64_t ldd;
  Factors f;
  int out_fp16;
  bool rows8;        // D's rows start on 8 bytes
  int M, N;          // rows of x, rows of the weight
  int ksteps, k_last;
  int bn;            // rows of x, up to a multiple of 32
  int stages, stage_bytes;
  int split, per_split;  // CTAs of a cluster, K steps of each
  int early;
  int* status;
};

__global__ void __launch_bounds__(kSmallThreads, 2)
int8_gemm_small_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ SmallParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ SmallBars sm;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = warp_id(), lane = lane_id();
  const int tw = blockIdx.x / p.split, rank = blockIdx.x % p.split;  // tile of the weight's rows, rank in the cluster
  const int k0 = rank * p.per_split, steps = max(0, min(p.ksteps, k0 + p.per_split) - k0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSmallStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.acc_full, 1);
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, kSmallBN);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      auto load_w = [&](int i, int s) {
        mbar_arrive_expect_tx(&sm.full[s], kABytes + p.bn * 128);
        tma_load_2d(ring + s * p.stage_bytes, &tm_w, &sm.full[s], (k0 + i) * kBK, tw * kBM);
      };
      auto load_x = [&](int i, int s) {
        tma_load_2d(ring + s * p.stage_bytes + kABytes, &tm_x, &sm.full[s], (k0 + i) * kBK, 0);
      };
      const int first = min(steps, p.stages);
      for (int i = 0; i < first; ++i) load_w(i, i);
      if (p.early) wait_for_previous_grid();
      for (int i = 0; i < first; ++i) load_x(i, i);
      int i = first, s = 0;
      uint32_t ph = 0;
      for (; i < steps; ++i) {
        if (!mbar_wait(&sm.empty[s], ph, kStatusTimeoutEmpty, abort_flag, p.status)) break;
        load_w(i, s);
        load_x(i, s);
        if (++s == p.stages) s = 0, ph ^= 1;
      }
      for (int j = max(0, i - p.stages); j < i; ++j)  // all copies land before the ring is used for the sums
        mbar_wait(&sm.full[j % p.stages], (j / p.stages) & 1, kStatusTimeoutTmaFull, nullptr, p.status);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the loop and one lane issues: the descriptors stay in uniform registers.
    const uint64_t da = smem_desc_sw128(smem_u32(ring), 16, 1024), db = smem_desc_sw128(smem_u32(ring) + kABytes, 16, 1024);
    const uint32_t idesc = idesc_of(Mma::kI8, kBM, p.bn, false, false);
    bool ok = true;
    int s = 0;  // the step's stage
    uint32_t ph = 0;
    for (int i = 0; i < steps; ++i) {
      ok = mbar_wait(&sm.full[s], ph, kStatusTimeoutTmaFull, abort_flag, p.status);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint64_t off = (uint64_t)(s * p.stage_bytes) >> 4;
      const int nk = k0 + i == p.ksteps - 1 ? p.k_last : 4;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (kk < nk) mma_ss<Mma::kI8, 1>(tmem, da + off + 2 * kk, db + off + 2 * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&sm.empty[s]);
      }
      __syncwarp();
      if (++s == p.stages) s = 0, ph ^= 1;
    }
    if (elect_one()) {
      if (!ok) *abort_flag = 1;
      mma_commit(&sm.acc_full);
      mbar_wait(&sm.acc_full, 0, kStatusTimeoutMma, nullptr, p.status);
    }
  } else {  // factors and biases of the weight rows, read while the operands come in
    const int r = threadIdx.x - 64, n = min(tw * kBM + r, p.N - 1);
    sm.col[r] = make_float2(__ldg(p.f.rb + n), p.f.bias.at(n));
  }
  // the MMAs are done and every copy has landed: the ring becomes the part's sums
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int* part = reinterpret_cast<int*>(ring);
  if (warp >= 2) {
    const int wq = warp & 3, row = wq * 32 + lane;
    const uint32_t acc = tmem + ((uint32_t)(wq * 32) << 16);
    for (int c = 0; c < p.bn; c += 32) {
      uint32_t r[32];
      tmem_ld32(acc + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 32; ++q) part[(c + q) * kBM + row] = steps > 0 ? (int)r[q] : 0;
    }
  }
  if (p.early) wait_for_previous_grid();  // the row factors of x are read below
  tc_fence_before();
  __syncthreads();
  if (p.split > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kSmallBN);
  }
  // this CTA's share of x's rows: a warp takes eight of them at a time (that many loads in flight), a lane four weight
  // rows of each
  const int per = (p.bn + p.split - 1) / p.split, c_end = min(p.M, (rank + 1) * per);
  constexpr int kWarps = kSmallThreads / 32, kRows = 8;
  const int n = tw * kBM + lane * 4;
  float2 cf[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) cf[q] = sm.col[lane * 4 + q];
  for (int c0 = rank * per + warp; c0 < c_end; c0 += kWarps * kRows) {
    int v[kRows][4];
#pragma unroll
    for (int u = 0; u < kRows; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[u][q] = 0;
    for (int r = 0; r < p.split; ++r) {
      const uint32_t from = p.split > 1 ? cluster_map(part + lane * 4, r) : smem_u32(part + lane * 4);
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int c = c0 + u * kWarps;
        if (c < c_end) {
          const float4 q = ld_cluster_float4(from + c * (kBM * 4));
          v[u][0] += __float_as_int(q.x);
          v[u][1] += __float_as_int(q.y);
          v[u][2] += __float_as_int(q.z);
          v[u][3] += __float_as_int(q.w);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int c = c0 + u * kWarps;
      if (c >= c_end || n >= p.N) continue;
      const float ra = p.f.ra[c];
      const bool far = far_out(ra);
      float y[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float s = __int2float_rn(v[u][q]);
        y[q] = far ? apply_factors_far(s, ra, cf[q].x, cf[q].y) : apply_factors(s, ra, cf[q].x, cf[q].y);
      }
      uint16_t* d = static_cast<uint16_t*>(p.d) + (int64_t)c * p.ldd + n;
      const uint32_t lo = p.out_fp16 ? pack16<true>(y[0], y[1]) : pack16<false>(y[0], y[1]);
      const uint32_t hi = p.out_fp16 ? pack16<true>(y[2], y[3]) : pack16<false>(y[2], y[3]);
      if (p.rows8) {
        *reinterpret_cast<uint2*>(d) = make_uint2(lo, hi);
      } else {
        d[0] = (uint16_t)lo;
        if (n + 1 < p.N) d[1] = (uint16_t)(lo >> 16);
        if (n + 2 < p.N) d[2] = (uint16_t)hi;
        if (n + 3 < p.N) d[3] = (uint16_t)(hi >> 16);
      }
    }
  }
  if (p.split > 1) {
    __syncthreads();
    cluster_sync();  // the other CTAs have read this one's part
  }
}

constexpr int kSmallSmem = 109 * 1024;  // dynamic shared memory of a CTA of the few-rows kernel: two fit an SM

CUtensorMap code_map(const Int8Matrix& x, uint32_t box_rows) {  // zeros past column K, whatever is stored there
  const uint64_t dims[2] = {(uint64_t)x.cols, (uint64_t)x.rows};
  const uint64_t strides[1] = {(uint64_t)x.row_bytes()};
  const uint32_t box[2] = {128u, box_rows};
  return make_tmap_u8(x.data, 2, dims, strides, box);
}

void launch_small(const Int8Matrix& a, const Int8Matrix& b, const Factors& f, at::Tensor& d, int device, cudaStream_t stream,
                  bool early) {
  const int sms = sm_count(device);
  SmallParams p;
  p.d = d.data_ptr();
  p.ldd = b.rows;
  p.f = f;
  p.out_fp16 = d.scalar_type() == at::kHalf ? 1 : 0;
  p.rows8 = (reinterpret_cast<uintptr_t>(p.d) | (uintptr_t)(2 * p.ldd)) % 8 == 0;
  p.M = (int)a.rows;
  p.N = (int)b.rows;
  p.ksteps = (int)((a.cols + kBK - 1) / kBK);
  p.k_last = (int)((a.cols - (int64_t)(p.ksteps - 1) * kBK + 31) / 32);
  p.bn = (p.M + 31) / 32 * 32;
  p.stage_bytes = kABytes + p.bn * 128;
  p.stages = std::min(kSmallStages, (kSmallSmem - 1024) / p.stage_bytes);
  // CTAs for up to four fifths of the places (two an SM): above that, and with clusters of more than six, they no longer
  // all run at once
  const int tiles = (p.N + kBM - 1) / kBM;
  p.split = std::max(1, std::min({6, sms * 2 * 4 / 5 / tiles, p.ksteps}));
  p.per_split = (p.ksteps + p.split - 1) / p.split;
  p.early = early ? 1 : 0;
  p.status = device_status_ptr(device);
  const CUtensorMap mw = code_map(b, kBM), mx = code_map(a, p.bn);
  // the ring, and the int32 sums that take its place
  const int smem = std::max(p.stages * p.stage_bytes, p.bn * kBM * 4) + 1024;
  raise_smem<int8_gemm_small_kernel>(kSmallSmem, device);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.split));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, int8_gemm_small_kernel, mw, mx, p));
}

template <bool FP16>
void launch_pair(const Int8Matrix& a, const Int8Matrix& b, const Factors& f, at::Tensor& d, int device, cudaStream_t stream,
                 bool early) {
  const int64_t M = a.rows, N = b.rows;
  PairGemm p = pair_gemm(M, N, a.cols, 1, false, false, device);
  p.early = early ? 1 : 0;
  p.b_old = 1;
  const CUtensorMap ma = code_map(a, kPairHalf), mb = code_map(b, kPairHalf);
  const OutRows out = out_rows(d.data_ptr(), N, M, N);
  const typename ScaleEpilogue<FP16>::Args args{out.tma ? out_rows_map(out) : ma, out, f};
  const at::Tensor parts = part_memory(p, d.options());
  launch_pair_gemm<Mma::kI8, ScaleEpilogue<FP16>>(ma, mb, parts, args, p, device, stream);
  if (p.split > 1)
    launch_overlapping(int8_part_sum_kernel<FP16>, part_grid(p), dim3(kPartThreads), 0, stream, true,
                       PartSum{parts.data_ptr<int>(), p, out, f});
}

template <typename T, bool ALIGNED>
void launch_vector_as(const VectorParams& p, int device, cudaStream_t stream) {
  // a row for each warp at least, and as many blocks as run at once
  const int grid = std::max(1, std::min(p.N / (kVectorThreads / 32), kVectorBlocks * sm_count(device)));
  const int smem = (int)((int8_row_bytes(p.K) + 511) / 512 * 512) + 4 * ((p.N + grid - 1) / grid);
  raise_smem<int8_vector_kernel<T, ALIGNED>>(kVectorSmem, device);
  int8_vector_kernel<T, ALIGNED><<<grid, kVectorThreads, smem, stream>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// One row, whose codes and the sums of a block's rows of the weight fit into shared memory.
bool one_row(int64_t M, const Int8Matrix& w, int device) {
  return M == 1 && w.cols <= kVectorMaxK && w.rows <= (int64_t)sm_count(device) * kVectorBlocks * kVectorMaxRows;
}

// d = x b^T + bias for one row x of 16 bits, or coded with the scale x_scale.
void launch_vector(const void* x, at::ScalarType type, const float* x_scale, const Int8Matrix& b,
                   const c10::optional<at::Tensor>& bias, at::Tensor& d, cudaStream_t stream) {
  if (b.rows == 0) return;
  const VectorParams p{x, b.data, d.data_ptr(), Factors{x_scale, b.row_scale, float_row(bias)}, d.scalar_type() == at::kHalf ? 1 : 0,
                 (int)b.rows, (int)b.cols};
  const bool aligned = b.cols % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 32 == 0;
  const int device = d.get_device();
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    if (aligned) launch_vector_as<T, true>(p, device, stream);
    else launch_vector_as<T, false>(p, device, stream);
  };
  if (type == at::kChar) launch_vector_as<int8_t, true>(p, device, stream);
  else if (type == at::kHalf) typed(__half{});
  else typed(__nv_bfloat16{});
}

// d [a.rows, b.rows] (bf16 or fp16, contiguous) = a b^T + bias, on the current device and stream.  early: the kernel before
// this one on the stream is the quantiser that wrote a, launched without overlap itself.
void gemm(const Int8Matrix& a, const Int8Matrix& b, const c10::optional<at::Tensor>& bias, at::Tensor& d, cudaStream_t stream,
          bool early) {
  if (a.rows == 0 || b.rows == 0) return;
  const Factors f{a.row_scale, b.row_scale, float_row(bias)};
  const int device = d.get_device();
  if (a.rows <= kSmallBN) launch_small(a, b, f, d, device, stream, early);
  else if (d.scalar_type() == at::kHalf) launch_pair<true>(a, b, f, d, device, stream, early);
  else launch_pair<false>(a, b, f, d, device, stream, early);
}

void check_sum(int64_t K) {
  DMAD_VALUE_CHECK(K <= kMaxK, "int8_linear: " + num(K) + " columns: int32 sums hold " + num(kMaxK) + " at most");
}

}  // namespace

// x W^T + bias for x [..., K] (bf16 or fp16), quantised here by rows, and W [N, K] stored in 8 bits by rows; the result in
// bf16 (0), fp16 (1) or x's type (-1).
at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& data, const at::Tensor& scale, c10::optional<at::Tensor> bias,
                       int64_t N, int64_t K, int64_t out_type) {
  const auto dt = x.scalar_type();
  DMAD_VALUE_CHECK(x.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf), "int8_linear: x must be bf16 or fp16 on CUDA");
  DMAD_VALUE_CHECK(x.dim() >= 1 && x.size(-1) == K, "int8_linear: x " + shape_text(x) + " must have " + num(K) + " columns");
  const Int8Matrix w = int8_matrix(data, scale, N, K, false, x.device(), "int8_linear: w");
  check_sum(K);
  const auto b = checked_bias(bias, N, x.device(), "int8_linear");
  c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor x2 = int8_rows(x, "int8_linear");
  Int8Matrix q{nullptr, nullptr, nullptr, x2.size(0), K};
  const auto plain = x.options().requires_grad(false);
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, plain.dtype(out_type == 0 ? at::kBFloat16 : out_type == 1 ? at::kHalf : dt));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (one_row(q.rows, w, y.get_device())) {
    launch_vector(x2.data_ptr(), dt, nullptr, w, b, y, stream);
    return y;
  }
  // codes and scales of x in one piece, freed to the stream's pool when the call returns
  const int64_t at_scales = (q.rows * q.row_bytes() + 511) / 512 * 512;
  at::Tensor work = at::empty({at_scales + 4 * q.rows}, plain.dtype(at::kByte));
  q.data = reinterpret_cast<int8_t*>(work.data_ptr());
  q.row_scale = reinterpret_cast<float*>(work.data_ptr<uint8_t>() + at_scales);
  int8_quantize_launch(x2, q, stream);
  gemm(q, w, b, y, stream, true);
  return y;
}

// The same for an x [M, K] that is stored in 8 bits by rows; the result [M, N] in bf16 (0) or fp16 (1).
at::Tensor int8_matmul(const at::Tensor& xdata, const at::Tensor& xscale, int64_t M, const at::Tensor& data,
                       const at::Tensor& scale, c10::optional<at::Tensor> bias, int64_t N, int64_t K, int64_t out_type) {
  DMAD_VALUE_CHECK(data.is_cuda(), "int8_linear: the native kernel takes CUDA tensors");
  const Int8Matrix w = int8_matrix(data, scale, N, K, false, data.device(), "int8_linear: w");
  const Int8Matrix q = int8_matrix(xdata, xscale, M, K, false, data.device(), "int8_linear: x");
  check_sum(K);
  const auto b = checked_bias(bias, N, data.device(), "int8_linear");
  c10::cuda::CUDAGuard guard(data.device());
  at::Tensor y = at::empty({M, N}, data.options().dtype(out_type == 1 ? at::kHalf : at::kBFloat16));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (one_row(M, w, y.get_device())) launch_vector(q.data, at::kChar, q.row_scale, w, b, y, stream);
  else gemm(q, w, b, y, stream, false);
  return y;
}

}  // namespace dmad
