// Persistent tcgen05 GEMM of block-scaled 4-bit operands for sm_100a.
//
//   D[M, N] = ra[m] rb[n] * sum_k A[m, k] B[n, k] + bias[n]          (bf16 or fp16 out, fp32 accumulation)
//
// A and B are e2m1 codes with one scale per 32 (mxfp4) or 16 (nvfp4) columns of K, multiplied on the tensor core
// (kind::mxf4 / kind::mxf4nvf4), ra / rb the nvfp4 row scales applied to the accumulator in the epilogue.
// The storage layout is described in fp4.cuh.
//
// Structure (one CTA per SM, persistent over 128 x 256 output tiles):
//   warp 0      producer: a ring of stages of 256 columns of K: A 128 x 128 bytes and B 256 x 128 bytes by TMA
//               (128-byte swizzle), and their scale tiles by plain bulk copies
//   warp 1      TMEM owner; one thread copies a stage's scale tiles to tensor memory (tcgen05.cp) and issues its
//               four K = 64 MMAs
//   warps 2..5  epilogue: tcgen05.ld (thread = output row), row scales, bias, stores
// Tensor memory: scales of a stage take up to 48 columns, double-buffered in the last 96 columns; the two 256-column
// accumulators overlap in columns [160, 256).  The epilogue drains the shared columns first and then releases the
// accumulator, so the next tile's MMAs start while five eighths of the tile are still being stored.
// Every mbarrier wait is bounded (2 s), records a status code and makes all roles leave.
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "common.cuh"
#include "fp4_host.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace dmad {

int* device_status_ptr(int device);
at::Tensor fp4_rows(const at::Tensor& x, const char* name);

namespace {

constexpr int kBM = 128, kBN = 256, kStages = 4;
constexpr int kBK = 256;                 // columns of K of a stage: 128 bytes of codes
constexpr int kABytes = kBM * 128;       // 16 KB
constexpr int kBBytes = kBN * 128;       // 32 KB
constexpr int kMaxTiles = 4;             // scale tiles along K of a stage (nvfp4; mxfp4 has two)
constexpr int kSaBytes = kMaxTiles * kFp4TileBytes;      // 2 KB
constexpr int kSbBytes = 2 * kMaxTiles * kFp4TileBytes;  // 4 KB
constexpr int kAcc1 = 160;               // first column of the second accumulator
constexpr int kSfCol = 416;              // first column of the scales
constexpr int kSfCols = 48;              // columns of one scale buffer

struct Smem {
  uint8_t a[kStages][kABytes];
  uint8_t b[kStages][kBBytes];
  uint8_t sa[kStages][kSaBytes];
  uint8_t sb[kStages][kSbBytes];
  float2 col[2][kBN];                  // row factor of B and bias of a tile's columns, by tile parity
  uint16_t stage[4][32][18];           // a warp's 32 rows x 16 columns on their way to unaligned rows of D
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[2], acc_free;
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};

struct Params {
  void* d;
  int64_t ldd;
  const uint8_t* sa;
  const uint8_t* sb;
  const float* ra;
  const float* rb;
  const void* bias;
  int bias_type;  // 0 fp32, 1 bf16, 2 fp16
  int out_fp16;
  int vec;        // bytes of a store: 32, 16 or 2, by the alignment of D's rows
  int M, N, K;
  int ktiles;     // scale tiles along K
  int ksteps;     // stages along K
  int tiles_m, tiles_n, num_tiles;
  int* status;
};

__device__ __forceinline__ float load_bias(const Params& p, int n) {
  if (p.bias_type == 0) return __ldg(static_cast<const float*>(p.bias) + n);
  if (p.bias_type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  return __half2float(static_cast<const __half*>(p.bias)[n]);
}

__device__ __forceinline__ uint32_t pack_out(const Params& p, float lo, float hi) {
  if (p.out_fp16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}

__device__ __forceinline__ void tile_coords(const Params& p, int t, int& tm, int& tn) {
  // column-major raster within groups of 8 M-tiles: neighbouring CTAs share B tiles in L2
  constexpr int kGroup = 8;
  const int group = t / (kGroup * p.tiles_n);
  const int first_m = group * kGroup;
  const int gm = min(kGroup, p.tiles_m - first_m);
  const int in = t % (kGroup * p.tiles_n);
  tm = first_m + in % gm;
  tn = in / gm;
}

// Stores 32 columns from nc of the warp's rows m0 .. m0 + 31 (o: the lane's row) to rows of D that are no multiple of
// 16 bytes: through shared memory, so that a warp still writes runs of 32 bytes.
__device__ __forceinline__ void store_unaligned(const Params& p, uint16_t (*stage)[18], int m0, int nc,
                                                const uint32_t (&o)[16]) {
  const int lane = lane_id();
  uint16_t* d0 = static_cast<uint16_t*>(p.d) + (int64_t)m0 * p.ldd + nc;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q) *reinterpret_cast<uint32_t*>(&stage[lane][2 * q]) = o[8 * h + q];
    __syncwarp();
    const int cc = lane & 15, n = 16 * h + cc;
    for (int r = lane >> 4; r < 32; r += 2)
      if (m0 + r < p.M && nc + n < p.N) d0[(int64_t)r * p.ldd + n] = stage[r][cc];
  }
}

// The same to any rows: whole 32-byte sectors where they allow it.
__device__ __forceinline__ void store_chunk(const Params& p, uint16_t (*stage)[18], uint16_t* drow, int m0, int nc,
                                            const uint32_t (&o)[16]) {
  const int lane = lane_id();
  if (p.vec == 32) {  // N % 16 == 0: a group of 16 columns is inside the row or past it
    if (m0 + lane < p.M) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (nc + 16 * q < p.N) st256(drow + nc + 16 * q, o + 8 * q);
    }
  } else if (p.vec == 16) {
    if (m0 + lane < p.M) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (nc + 8 * q < p.N)
          *reinterpret_cast<uint4*>(drow + nc + 8 * q) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
    }
  } else {
    store_unaligned(p, stage, m0, nc, o);
  }
}

template <bool NV>
__global__ void __launch_bounds__(192, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = warp_id(), lane = lane_id();
  constexpr int kStageTiles = NV ? 4 : 2;  // scale tiles along K of a whole stage

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.acc_full[0], 1);
    mbar_init(&sm.acc_full[1], 1);
    mbar_init(&sm.acc_free, 128);
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int it = 0;  // global stage counter (ring position)
      bool ok = true;
      const int sb_rows = (p.N + kFp4TileRows - 1) / kFp4TileRows;
      for (int t = blockIdx.x; ok && t < p.num_tiles; t += gridDim.x) {
        int tm, tn;
        tile_coords(p, t, tm, tn);
        const bool second = tn * 2 + 1 < sb_rows;  // whether B's tile has rows in a second scale tile
        for (int k = 0; k < p.ksteps; ++k, ++it) {
          const int s = it % kStages;
          const uint32_t ph = (it / kStages) & 1;
          if (!(ok = mbar_wait(&sm.empty[s], ph ^ 1, kStatusTimeoutEmpty, abort_flag, p.status))) break;
          const int kt = k * kStageTiles;
          const uint32_t bytes = (uint32_t)min(kStageTiles, p.ktiles - kt) * kFp4TileBytes;
          mbar_arrive_expect_tx(&sm.full[s], kABytes + kBBytes + bytes * (second ? 3 : 2));
          tma_load_2d(sm.a[s], &tm_a, &sm.full[s], k * 128, tm * kBM);
          tma_load_2d(sm.b[s], &tm_b, &sm.full[s], k * 128, tn * kBN);
          bulk_load(sm.sa[s], p.sa + ((int64_t)tm * p.ktiles + kt) * kFp4TileBytes, bytes, &sm.full[s]);
          const uint8_t* sb = p.sb + ((int64_t)(2 * tn) * p.ktiles + kt) * kFp4TileBytes;
          bulk_load(sm.sb[s], sb, bytes, &sm.full[s]);
          if (second) bulk_load(sm.sb[s] + kSaBytes, sb + (int64_t)p.ktiles * kFp4TileBytes, bytes, &sm.full[s]);
        }
      }
      // all issued copies land before the CTA's shared memory goes away
      for (int j = max(0, it - kStages); j < it; ++j)
        mbar_wait(&sm.full[j % kStages], (j / kStages) & 1, kStatusTimeoutTmaFull, nullptr, p.status);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      int it = 0, tl = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < p.num_tiles; t += gridDim.x, ++tl) {
        // the columns shared with the previous tile's accumulator have been drained
        if (tl > 0 && !(ok = mbar_wait(&sm.acc_free, (tl - 1) & 1, kStatusTimeoutSoftmax, abort_flag, p.status))) break;
        tc_fence_after();
        const uint32_t d = tmem + ((tl & 1) ? kAcc1 : 0);
        for (int k = 0; k < p.ksteps; ++k, ++it) {
          const int s = it % kStages;
          if (!(ok = mbar_wait(&sm.full[s], (it / kStages) & 1, kStatusTimeoutTmaFull, abort_flag, p.status))) break;
          // this stage's scale buffer was last read by the MMAs of two stages ago
          if (it >= 2 && !(ok = mbar_wait(&sm.empty[(it - 2) % kStages], ((it - 2) / kStages) & 1, kStatusTimeoutMma,
                                          abort_flag, p.status)))
            break;
          tc_fence_after();
          const uint32_t sfa = tmem + kSfCol + (it & 1) * kSfCols, sfb = sfa + 16;
          const int nt = min(kStageTiles, p.ktiles - k * kStageTiles);
          const uint32_t aa = smem_u32(sm.a[s]), bb = smem_u32(sm.b[s]);
          const uint32_t ssa = smem_u32(sm.sa[s]), ssb = smem_u32(sm.sb[s]);
          for (int j = 0; j < nt; ++j) {
            tmem_cp_scales<1>(sfa + 4 * j, smem_desc_scales(ssa + j * kFp4TileBytes));
            tmem_cp_scales<1>(sfb + 8 * j, smem_desc_scales(ssb + j * kFp4TileBytes));
            tmem_cp_scales<1>(sfb + 8 * j + 4, smem_desc_scales(ssb + kSaBytes + j * kFp4TileBytes));
          }
          const int nk = min(4, (p.K - k * kBK + 63) / 64);
          for (int kk = 0; kk < nk; ++kk) {
            const int j = NV ? kk : kk >> 1;
            const uint32_t idesc = idesc_fp4(NV, kBM, kBN, NV ? 0 : (kk & 1) * 2);
            mma_fp4_ss<NV, 1>(d, smem_desc_sw128(aa + kk * 32, 16, 1024), smem_desc_sw128(bb + kk * 32, 16, 1024), idesc,
                           sfa + 4 * j, sfb + 8 * j, (k > 0 || kk > 0) ? 1u : 0u);
          }
          mma_commit(&sm.empty[s]);
        }
        if (!ok) break;
        mma_commit(&sm.acc_full[tl & 1]);
      }
      if (!ok) *abort_flag = 1;
      mma_commit(&sm.drain);
      mbar_wait(&sm.drain, 0, kStatusTimeoutMma, nullptr, p.status);
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..5)
    const int wq = warp & 3;  // TMEM lane quarter this warp may access
    const int row = wq * 32 + lane;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const int et = threadIdx.x - 64;
    int tl = 0;
    for (int t = blockIdx.x; t < p.num_tiles; t += gridDim.x, ++tl) {
      int tm, tn;
      tile_coords(p, t, tm, tn);
      const int m = tm * kBM + row;
      // the tile's column factors and biases, read while its MMAs run (a buffer is written again only after
      // the barrier of the tile in between)
      float2* col = sm.col[tl & 1];
#pragma unroll
      for (int i = et; i < kBN; i += 128) {
        const int n = min(tn * kBN + i, p.N - 1);
        col[i] = make_float2(NV ? __ldg(p.rb + n) : 1.f, p.bias != nullptr ? load_bias(p, n) : 0.f);
      }
      const float ra = (NV && m < p.M) ? __ldg(p.ra + m) : 1.f;
      const bool ok = mbar_wait(&sm.acc_full[tl & 1], (tl >> 1) & 1, kStatusTimeoutMma, abort_flag, p.status);
      // also the barrier of the column factors; all four warps leave together, since it counts them
      if (named_bar_any(1, 128, !ok)) break;
      tc_fence_after();
      uint16_t* drow = static_cast<uint16_t*>(p.d) + (int64_t)m * p.ldd;
      const uint32_t acc = tmem + lane_base + ((tl & 1) ? kAcc1 : 0);
      // chunks of 32 columns, the ones shared with the other accumulator first: the last three of the
      // first accumulator, the first three of the second
#pragma unroll 1
      for (int i = 0; i < kBN / 32; ++i) {
        const int c = (tl & 1) ? i : (i < 3 ? 5 + i : i - 3);
        uint32_t r[32];
        tmem_ld32(acc + c * 32, r);
        tmem_wait_ld();
        if (i == 2) {
          tc_fence_before();
          mbar_arrive(&sm.acc_free);
        }
        const int nc = tn * kBN + c * 32;
        if (nc >= p.N) continue;
        uint32_t o[16];
        const float4* cf = reinterpret_cast<const float4*>(col + c * 32);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float4 f = cf[q];
          o[q] = pack_out(p, fmaf(__uint_as_float(r[2 * q]) * ra, f.x, f.y),
                          fmaf(__uint_as_float(r[2 * q + 1]) * ra, f.z, f.w));
        }
        store_chunk(p, sm.stage[wq], drow, m - lane, nc, o);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- CTA pairs
// The same product with a pair of CTAs on each 256 x 256 tile (cta_group::2): each CTA holds 128 rows of A and of D and
// loads 128 of B's 256 rows, so a stage moves 38 KB into an SM instead of 54 KB and the L2 is read a third less.
//   warp 0      producer of its own CTA's operands and scales (all of B's scales: each CTA multiplies all of B), which
//               all complete on the leader's barriers
//   warp 1      leader CTA: the MMA thread, which also copies the scales of both CTAs to tensor memory.  A copy takes
//               some 56 cycles of the tensor core's queue and a stage has 12 (nvfp4) or 6 (mxfp4), so the next
//               stage's copies are issued between this stage's MMAs, where they run beside them
//   warps 2..9  epilogue of the CTA's 128 rows: two warps a lane quarter, every other 32 columns each; rows leave
//               through shared memory by TMA (direct stores of a lane's row cost the SM four times the cycles)
// Tensor memory: scale buffers in the last 144 columns (three of 48 for nvfp4, six of 24 for mxfp4), accumulators at 0
// and 112.  The epilogue reads the 144 shared columns into registers at once and then releases the accumulator.
constexpr int kPairBM = 256, kPairStages = 5;
constexpr int kPairAcc1 = 112, kPairSfCol = 368;
constexpr int kEpiWarps = 8, kPairThreads = 64 + 32 * kEpiWarps;

struct PairSmem {
  uint8_t a[kPairStages][kABytes];
  uint8_t b[kPairStages][kABytes];
  uint8_t sa[kPairStages][kSaBytes];
  uint8_t sb[kPairStages][kSbBytes];
  uint8_t stage[kEpiWarps][2048];  // a warp's 32 rows x 32 columns of D on their way out
  float2 col[2][kBN];
  uint64_t full[kPairStages], empty[kPairStages];
  uint64_t acc_full[2], acc_free;
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <bool NV>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                     const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb,
                     const __grid_constant__ CUtensorMap tm_d, Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  PairSmem& sm = *reinterpret_cast<PairSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  constexpr int kStageTiles = NV ? 4 : 2;          // scale tiles along K of a whole stage
  constexpr int kSfBufCols = 12 * kStageTiles;     // A: 4 columns a tile, B: 8
  constexpr int kSfBufs = 144 / kSfBufCols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&sm.full[s], 1);  // the leader's counts both CTAs' bytes; the other CTA's is not used
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.acc_full[0], 1);
    mbar_init(&sm.acc_full[1], 1);
    mbar_init(&sm.acc_free, 2 * kEpiWarps);
    mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&sm.tmem_base, 512);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_sa);
    prefetch_tmap(&tm_sb);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      const int sa_rows = (p.M + kFp4TileRows - 1) / kFp4TileRows, sb_rows = (p.N + kFp4TileRows - 1) / kFp4TileRows;
      for (int t = cluster; ok && t < p.num_tiles; t += clusters) {
        int tm, tn;
        tile_coords(p, t, tm, tn);
        // scale tiles past the matrix do not exist; their rows are zeros in A and B and are not stored from D
        const int ra = tm * 2 + (int)rank;
        const bool second = tn * 2 + 1 < sb_rows;
        const uint32_t scale_boxes = (tm * 2 + 1 < sa_rows ? 2 : 1) + (second ? 4 : 2);  // of both CTAs
        for (int k = 0; k < p.ksteps; ++k, ++it) {
          const int s = it % kPairStages;
          const uint32_t ph = (it / kPairStages) & 1;
          if (!(ok = mbar_wait(&sm.empty[s], ph ^ 1, kStatusTimeoutEmpty, abort_flag, p.status))) break;
          // a box is written, and counted, whole: columns past K and scale tiles past the last are zeros
          constexpr uint32_t box = kStageTiles * kFp4TileBytes;
          if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], 4 * kABytes + box * scale_boxes);
          const uint32_t full = cluster_map(&sm.full[s], 0);
          const int kt = k * kStageTiles * (kFp4TileBytes / 8);
          tma_load_2d_pair(sm.a[s], &tm_a, full, k * 128, ra * kBM);
          tma_load_2d_pair(sm.b[s], &tm_b, full, k * 128, (tn * 2 + (int)rank) * kBM);
          if (ra < sa_rows) tma_load_2d_pair(sm.sa[s], &tm_sa, full, kt, ra);
          tma_load_2d_pair(sm.sb[s], &tm_sb, full, kt, 2 * tn);
          if (second) tma_load_2d_pair(sm.sb[s] + kSaBytes, &tm_sb, full, kt, 2 * tn + 1);
        }
      }
      // all issued copies land before a CTA's shared memory goes away
      if (rank == 0)
        for (int j = max(0, it - kPairStages); j < it; ++j)
          mbar_wait_cluster(&sm.full[j % kPairStages], (j / kPairStages) & 1, kStatusTimeoutTmaFull, nullptr, p.status);
    }
  } else if (warp == 1 && rank != 0) {
    // the leader issues the pair's MMAs
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (elect_one()) {
      const int my_tiles = cluster < p.num_tiles ? (p.num_tiles - 1 - cluster) / clusters + 1 : 0;
      const int total = my_tiles * p.ksteps;  // stages of all tiles
      bool ok = true;
      // waits for stage i's operands and for its scale buffer, last read by the MMAs of kSfBufs stages before (with
      // as many buffers as stages the ring itself has waited for those)
      auto stage_ready = [&](int i) {
        return mbar_wait_cluster(&sm.full[i % kPairStages], (i / kPairStages) & 1, kStatusTimeoutTmaFull, abort_flag,
                                 p.status) &&
               (kSfBufs >= kPairStages || i < kSfBufs ||
                mbar_wait(&sm.empty[(i - kSfBufs) % kPairStages], ((i - kSfBufs) / kPairStages) & 1, kStatusTimeoutMma,
                          abort_flag, p.status));
      };
      auto stage_there = [&](int i) {  // the same without waiting
        return mbar_try_wait(smem_u32(&sm.full[i % kPairStages]), (i / kPairStages) & 1) &&
               (kSfBufs >= kPairStages || i < kSfBufs ||
                mbar_try_wait(smem_u32(&sm.empty[(i - kSfBufs) % kPairStages]), ((i - kSfBufs) / kPairStages) & 1));
      };
      // scale tile j along K of stage i, to tensor memory
      auto copy_scales = [&](int i, int j) {
        const int s = i % kPairStages;
        const uint32_t sfa = tmem + kPairSfCol + (i % kSfBufs) * kSfBufCols, sfb = sfa + 4 * kStageTiles;
        tmem_cp_scales<2>(sfa + 4 * j, smem_desc_scales(smem_u32(sm.sa[s]) + j * kFp4TileBytes));
        tmem_cp_scales<2>(sfb + 8 * j, smem_desc_scales(smem_u32(sm.sb[s]) + j * kFp4TileBytes));
        tmem_cp_scales<2>(sfb + 8 * j + 4, smem_desc_scales(smem_u32(sm.sb[s]) + kSaBytes + j * kFp4TileBytes));
      };
      auto scale_tiles = [&](int k) { return min(kStageTiles, p.ktiles - k * kStageTiles); };
      int it = 0;
      bool copied = false;  // this stage's scales are on their way already
      for (int tl = 0; ok && tl < my_tiles; ++tl) {
        // both CTAs have read the columns shared with the previous tile's accumulator
        if (tl > 0 &&
            !(ok = mbar_wait_cluster(&sm.acc_free, (tl - 1) & 1, kStatusTimeoutSoftmax, abort_flag, p.status)))
          break;
        tc_fence_after();
        const uint32_t d = tmem + ((tl & 1) ? kPairAcc1 : 0);
        for (int k = 0; k < p.ksteps; ++k, ++it) {
          const int s = it % kPairStages;
          if (!copied) {
            if (!(ok = stage_ready(it))) break;
            tc_fence_after();
            for (int j = 0; j < scale_tiles(k); ++j) copy_scales(it, j);
          }
          const int knext = k + 1 < p.ksteps ? k + 1 : 0;
          const int next_tiles = it + 1 < total && stage_there(it + 1) ? scale_tiles(knext) : 0;
          tc_fence_after();
          const uint32_t sfa = tmem + kPairSfCol + (it % kSfBufs) * kSfBufCols, sfb = sfa + 4 * kStageTiles;
          const uint32_t aa = smem_u32(sm.a[s]), bb = smem_u32(sm.b[s]);
          const int nk = min(4, (p.K - k * kBK + 63) / 64);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int j = NV ? kk : kk >> 1;
            const uint32_t idesc = idesc_fp4(NV, kPairBM, kBN, NV ? 0 : (kk & 1) * 2);
            if (kk < nk)
              mma_fp4_ss<NV, 2>(d, smem_desc_sw128(aa + kk * 32, 16, 1024), smem_desc_sw128(bb + kk * 32, 16, 1024),
                                idesc, sfa + 4 * j, sfb + 8 * j, (k > 0 || kk > 0) ? 1u : 0u);
            if (kk < next_tiles) copy_scales(it + 1, kk);
          }
          copied = next_tiles > 0;
          mma_commit_pair(&sm.empty[s]);
        }
        if (!ok) break;
        mma_commit_pair(&sm.acc_full[tl & 1]);
      }
      if (!ok) *abort_flag = 1;
      mma_commit_pair(&sm.drain);
      mbar_wait(&sm.drain, 0, kStatusTimeoutMma, nullptr, p.status);
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..9)
    const int ew = warp - 2, wq = warp & 3, half = ew >> 2;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const int et = threadIdx.x - 64;
    const uint32_t acc_free = cluster_map(&sm.acc_free, 0);
    uint8_t* stage = sm.stage[ew];
    // row of the warp's first lane, first column, and the factors of one tile
    int m0 = 0, n0 = 0;
    float ra = 1.f;
    float2 cf = make_float2(1.f, 0.f);
    auto fetch = [&](int t) {
      int tm, tn;
      tile_coords(p, t, tm, tn);
      m0 = tm * kPairBM + (int)rank * kBM + wq * 32;
      n0 = tn * kBN;
      const int n = min(n0 + et, p.N - 1);
      cf = make_float2(NV ? __ldg(p.rb + n) : 1.f, p.bias != nullptr ? load_bias(p, n) : 0.f);
      ra = (NV && m0 + lane < p.M) ? __ldg(p.ra + m0 + lane) : 1.f;
    };
    if (cluster < p.num_tiles) {
      fetch(cluster);
      sm.col[0][et] = cf;
    }
    int tl = 0;
    for (int t = cluster; t < p.num_tiles; t += clusters, ++tl) {
      const float2* col = sm.col[tl & 1];
      const int tm0 = m0, tn0 = n0;
      const float tra = ra;
      const bool ok = mbar_wait(&sm.acc_full[tl & 1], (tl >> 1) & 1, kStatusTimeoutMma, abort_flag, p.status);
      // also the barrier of the column factors; all warps leave together, since it counts them
      if (named_bar_any(1, 32 * kEpiWarps, !ok)) break;
      tc_fence_after();
      const uint32_t acc = tmem + lane_base + ((tl & 1) ? kPairAcc1 : 0);
      // order of the 32-column chunks: the five that share columns with the other accumulator first (3..7 of the
      // first, 0..4 of the second); this warp takes every other one
      const int shift = (tl & 1) ? 0 : 3;
      auto chunk = [&](int i) { return (2 * i + half + shift) & 7; };
      uint32_t r[3][32];
#pragma unroll
      for (int i = 0; i < 3; ++i) tmem_ld32(acc + chunk(i) * 32, r[i]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_free);
      // the next tile's factors are read while this tile is stored (all warps are past the tile before, whose
      // buffer they go to)
      if (t + clusters < p.num_tiles) fetch(t + clusters);
      auto finish = [&](int c, const uint32_t (&v)[32]) {
        const int nc = tn0 + c * 32;
        if (nc >= p.N || tm0 >= p.M) return;
        uint32_t o[16];
        const float4* f4 = reinterpret_cast<const float4*>(col + c * 32);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float4 f = f4[q];
          o[q] = pack_out(p, fmaf(__uint_as_float(v[2 * q]) * tra, f.x, f.y),
                          fmaf(__uint_as_float(v[2 * q + 1]) * tra, f.z, f.w));
        }
        if (p.vec >= 16) {  // rows of D are multiples of 16 bytes: a box of 32 x 32 by TMA, 64-byte swizzle
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&tm_d, stage, nc, tm0);
        } else {
          store_unaligned(p, reinterpret_cast<uint16_t(*)[18]>(stage), tm0, nc, o);
        }
      };
      finish(chunk(0), r[0]);
      tmem_ld32(acc + chunk(3) * 32, r[0]);
      finish(chunk(1), r[1]);
      finish(chunk(2), r[2]);
      tmem_wait_ld();
      finish(chunk(3), r[0]);
      sm.col[(tl + 1) & 1][et] = cf;
    }
    if (lane == 0) tma_store_wait_read();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the pair's barriers and tensor memory are no longer in use by the other CTA
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

CUtensorMap code_map(const Fp4Matrix& x, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t)x.row_bytes(), (uint64_t)x.rows};
  const uint64_t strides[1] = {(uint64_t)x.row_bytes()};
  const uint32_t box[2] = {128u, box_rows};
  return make_tmap_u8(x.data, 2, dims, strides, box);
}

// Raises a kernel's dynamic shared memory limit, once a device.
template <auto Kernel>
void configure(int smem, int device) {
  static std::array<std::atomic<bool>, 64> done{};
  if (device < 64 && done[device].load(std::memory_order_acquire)) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (device < 64) done[device].store(true, std::memory_order_release);
}

// Scales as a matrix of 8-byte elements, a row for each 128 rows of x, read in boxes of a stage's tiles.
CUtensorMap scale_map(const Fp4Matrix& x) {
  const uint64_t dims[2] = {(uint64_t)x.ktiles() * kFp4TileBytes / 8, (uint64_t)x.row_tiles()};
  const uint64_t strides[1] = {(uint64_t)x.ktiles() * kFp4TileBytes};
  const uint32_t box[2] = {(x.nv ? 4u : 2u) * kFp4TileBytes / 8, 1u};
  return make_tmap(CU_TENSOR_MAP_DATA_TYPE_FLOAT64, x.scales, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// D in boxes of 32 x 32, swizzled over 64 bytes in shared memory.
CUtensorMap out_map(const Params& p) {
  const uint64_t dims[2] = {(uint64_t)p.N, (uint64_t)p.M};
  const uint64_t strides[1] = {(uint64_t)p.ldd * 2};
  const uint32_t box[2] = {32u, 32u};
  return make_tmap_bf16(p.d, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <bool NV>
void launch(const Fp4Matrix& a, const Fp4Matrix& b, Params& p, int device, cudaStream_t stream) {
  const int sms = sm_count(device);
  if (p.M > 256) {
    p.tiles_m = (p.M + kPairBM - 1) / kPairBM;
    p.num_tiles = p.tiles_m * p.tiles_n;
    const int smem = (int)sizeof(PairSmem) + 1024;
    const CUtensorMap ma = code_map(a, kBM), mb = code_map(b, kBM), sa = scale_map(a), sb = scale_map(b);
    configure<fp4_gemm_pair_kernel<NV>>(smem, device);
    fp4_gemm_pair_kernel<NV><<<2 * std::min(p.num_tiles, sms / 2), kPairThreads, smem, stream>>>(
        ma, mb, sa, sb, p.vec >= 16 ? out_map(p) : ma, p);
  } else {
    const int smem = (int)sizeof(Smem) + 1024;
    configure<fp4_gemm_kernel<NV>>(smem, device);
    fp4_gemm_kernel<NV><<<std::min(p.num_tiles, sms), 192, smem, stream>>>(code_map(a, kBM), code_map(b, kBN), p);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// d [a.rows, b.rows] (bf16 or fp16, contiguous) = a b^T + bias, on the current device and stream.
void gemm(const Fp4Matrix& a, const Fp4Matrix& b, const c10::optional<at::Tensor>& bias, at::Tensor& d,
          cudaStream_t stream) {
  const int64_t M = a.rows, N = b.rows, K = a.cols;
  if (M == 0 || N == 0) return;
  Params p;
  p.bias = nullptr;
  p.bias_type = 0;
  if (bias.has_value() && bias->defined()) {
    p.bias = bias->data_ptr();
    p.bias_type = bias->scalar_type() == at::kFloat ? 0 : bias->scalar_type() == at::kBFloat16 ? 1 : 2;
  }
  p.d = d.data_ptr();
  p.ldd = N;
  p.sa = a.scales;
  p.sb = b.scales;
  p.ra = a.row_scale;
  p.rb = b.row_scale;
  p.out_fp16 = d.scalar_type() == at::kHalf ? 1 : 0;
  const uintptr_t align = reinterpret_cast<uintptr_t>(p.d) | (uintptr_t)(2 * N);
  p.vec = align % 32 == 0 ? 32 : align % 16 == 0 ? 16 : 2;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.ktiles = (int)a.ktiles();
  p.ksteps = (int)((K + kBK - 1) / kBK);
  p.tiles_m = (int)((M + kBM - 1) / kBM);
  p.tiles_n = (int)((N + kBN - 1) / kBN);
  DMAD_VALUE_CHECK((int64_t)p.tiles_m * p.tiles_n <= INT32_MAX, "fp4_linear: too many output tiles");
  p.num_tiles = p.tiles_m * p.tiles_n;
  const int device = d.get_device();
  p.status = device_status_ptr(device);
  a.nv ? launch<true>(a, b, p, device, stream) : launch<false>(a, b, p, device, stream);
}

c10::optional<at::Tensor> checked_bias(const c10::optional<at::Tensor>& bias, int64_t N, const at::Device& device) {
  if (!(bias.has_value() && bias->defined())) return c10::nullopt;
  DMAD_VALUE_CHECK(bias->device() == device && bias->dim() == 1 && bias->size(0) == N && is_float_type(bias->scalar_type()),
                   "fp4_linear: bias must be bf16, fp16 or fp32 (" + num(N) + ",) on the device of w, got " +
                       dtype_name(bias->scalar_type()) + " " + shape_text(*bias));
  return bias->contiguous();
}

}  // namespace

// x W^T + bias for x [..., K] (bf16 or fp16), quantised here, and W [N, K] stored in 4 bits; the result in bf16 (0),
// fp16 (1) or x's type (-1).
at::Tensor fp4_linear(const at::Tensor& x, const at::Tensor& data, const at::Tensor& scales,
                      c10::optional<at::Tensor> row_scale, c10::optional<at::Tensor> bias, int64_t N, int64_t K, bool nv,
                      int64_t out_type) {
  const auto dt = x.scalar_type();
  DMAD_VALUE_CHECK(x.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf), "fp4_linear: x must be bf16 or fp16 on CUDA");
  DMAD_VALUE_CHECK(x.dim() >= 1 && x.size(-1) == K, "fp4_linear: x " + shape_text(x) + " must have " + num(K) + " columns");
  const Fp4Matrix w = fp4_matrix(data, scales, row_scale, N, K, nv, x.device(), "fp4_linear: w");
  const auto b = checked_bias(bias, N, x.device());
  const at::Tensor x2 = fp4_rows(x, "fp4_linear");
  Fp4Matrix q{nullptr, nullptr, nullptr, x2.size(0), K, nv};
  DMAD_VALUE_CHECK(q.rows <= INT32_MAX - 256, "fp4_linear: sizes out of range");
  c10::cuda::CUDAGuard guard(x.device());
  // codes, scales and row factors of x in one piece, freed to the stream's pool when the call returns
  const int64_t at_scales = (q.data_bytes() + 511) / 512 * 512, at_rows = at_scales + q.scale_bytes();
  const auto plain = x.options().requires_grad(false);
  at::Tensor work = at::empty({at_rows + (nv ? 4 * q.rows : 0)}, plain.dtype(at::kByte));
  q.data = work.data_ptr<uint8_t>();
  q.scales = q.data + at_scales;
  q.row_scale = nv ? reinterpret_cast<float*>(q.data + at_rows) : nullptr;
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, plain.dtype(out_type == 0 ? at::kBFloat16 : out_type == 1 ? at::kHalf : dt));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  fp4_quantize_launch(x2, q, stream);
  gemm(q, w, b, y, stream);
  return y;
}

// The same for an x [M, K] that is stored in 4 bits; the result [M, N] in bf16 (0) or fp16 (1).
at::Tensor fp4_matmul(const at::Tensor& xdata, const at::Tensor& xscales, c10::optional<at::Tensor> xrow_scale,
                      int64_t M, const at::Tensor& data, const at::Tensor& scales, c10::optional<at::Tensor> row_scale,
                      c10::optional<at::Tensor> bias, int64_t N, int64_t K, bool nv, int64_t out_type) {
  DMAD_VALUE_CHECK(data.is_cuda(), "fp4_linear: the native kernel takes CUDA tensors");
  const Fp4Matrix w = fp4_matrix(data, scales, row_scale, N, K, nv, data.device(), "fp4_linear: w");
  const Fp4Matrix q = fp4_matrix(xdata, xscales, xrow_scale, M, K, nv, data.device(), "fp4_linear: x");
  const auto b = checked_bias(bias, N, data.device());
  c10::cuda::CUDAGuard guard(data.device());
  at::Tensor y = at::empty({M, N}, data.options().dtype(out_type == 1 ? at::kHalf : at::kBFloat16));
  gemm(q, w, b, y, at::cuda::getCurrentCUDAStream());
  return y;
}

}  // namespace dmad
