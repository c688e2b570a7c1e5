// tcgen05 GEMMs of block-scaled 4-bit operands for sm_100a.
//
//   D[M, N] = ra[m] rb[n] * sum_k A[m, k] B[n, k] + bias[n]          (bf16 or fp16 out, fp32 accumulation)
//
// A and B are e2m1 codes with one scale per 32 (mxfp4) or 16 (nvfp4) columns of K, multiplied on the tensor core
// (kind::mxf4 / kind::mxf4nvf4), ra / rb the nvfp4 row scales applied to the accumulator in the epilogue, and one
// rounding at the end.  The storage layout is described in fp4.cuh.  Two kernels: pairs of CTAs on 256 x 256 tiles, and
// one for few rows (few_rows() says which).
//
// Both step through K in stages of 256 columns (128 bytes of a row): codes by TMA with a 128-byte swizzle, scale tiles to
// shared memory and from there by tcgen05.cp to tensor memory, then four K = 64 MMAs (fewer at the end of K).
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

constexpr int kBM = 128, kBN = 256;
constexpr int kBK = 256;            // columns of K of a stage: 128 bytes of codes
constexpr int kABytes = kBM * 128;  // 16 KB
constexpr int kMaxTiles = 4;        // scale tiles along K of a stage (nvfp4; mxfp4 has two)
constexpr int kSaBytes = kMaxTiles * kFp4TileBytes;      // 2 KB
constexpr int kSbBytes = 2 * kMaxTiles * kFp4TileBytes;  // 4 KB

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
  bool rows16;    // D's rows start on 16 bytes (and N is a multiple of 8)
  int M, N, K;
  int ktiles;     // scale tiles along K
  int ksteps;     // stages along K
  int tiles_m, tiles_n, num_tiles;  // of the pair kernel
  int* status;
};

__device__ __forceinline__ float load_bias(const Params& p, int n) {
  if (p.bias_type == 0) return __ldg(static_cast<const float*>(p.bias) + n);
  if (p.bias_type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  return __half2float(static_cast<const __half*>(p.bias)[n]);
}

template <bool FP16>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if constexpr (FP16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}

// acc ra rb + bias for nvfp4's factors of the row and of the column, without an overflow or a lost digit where the result
// has none.  An accumulator is 0 or of a size from 2^-20 (two codes and two scales) to 2^47 (K <= 2^24 products of at
// most (6 * 448)^2), so acc ra is an ordinary number for ra from 2^-80 to 2^80 and the last step rounds once.  For rows
// further out (elements above 1e27, or all below 1e-20) rb comes first, on acc c with c = 2^+-64, and ra / c last: acc c rb
// is larger than fp32 only if the result is, and small enough to lose digits only if the result is below 2^-140.
__device__ __forceinline__ bool far_out(float ra) { return !(ra >= 0x1p-80f && ra <= 0x1p80f); }
__device__ __forceinline__ float apply_factors(float acc, float ra, float rb, float bias) {
  return fmaf(acc * ra, rb, bias);
}
__device__ __forceinline__ float apply_factors_far(float acc, float ra, float rb, float bias) {
  const bool big = ra > 1.f;
  return fmaf(acc * (big ? 0x1p64f : 0x1p-64f) * rb, ra * (big ? 0x1p-64f : 0x1p64f), bias);
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
// 16 bytes: through shared memory, so that a warp still writes runs of 32 bytes.  (8192 x 8191 x 1536 mxfp4: 118 us, 58
// with 8192 columns; words of 4 bytes, shifted in every other row, 146 to 166 us.)
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

// ---------------------------------------------------------------- CTA pairs
// A pair of CTAs on each 256 x 256 tile (cta_group::2), persistent, one CTA an SM: each CTA holds 128 rows of A and of D
// and loads 128 of B's 256 rows, so a stage moves 38 KB into an SM (one CTA with a 128 x 256 tile: 54 KB, more than the
// some 64 bytes a cycle that the L2 gives an SM in the time of its MMAs).
//   warp 0      producer of its own CTA's operands and scales (all of B's scales: each CTA multiplies all of B), which
//               all complete on the leader's barriers
//   warp 1      leader CTA: issues the MMAs, and before them the copies of both CTAs' scales to tensor memory
//   warps 2..9  epilogue of the CTA's 128 rows: two warps a lane quarter, every other 32 columns each; rows leave
//               through shared memory by TMA (direct stores of a lane's row cost the SM four times the cycles)
// Tensor memory: scale buffers in the last 144 columns (three of 48 for nvfp4, six of 24 for mxfp4), accumulators at 0
// and 112.  The epilogue reads the 144 shared columns into registers at once and then releases the accumulator.
// Measured, two passes after a pause and 3 s of passes at the power limit: 37966 x 30720 x 5120 nvfp4 2.43 to 2.50 ms (4.9
// PFLOP/s) and 2.81 ms at 1.40 GHz, mxfp4 2.07 to 2.13 ms (5.7 PFLOP/s) and 2.41 ms at 1.24 GHz.  In cycles bound by the
// tensor core's queue, where a scale copy holds up the MMAs behind it for some 40 (nvfp4 has twelve a stage beside four
// MMAs, mxfp4 six); the clock is what the power limit leaves.  32760 x 8960 x 1536 mxfp4 0.22 ms, nvfp4 0.24 ms, where six
// stages of K are shorter than the epilogue of the tile.
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

template <bool NV, bool FP16>
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
      // and so do the leader's arrivals for the last stages, which nobody else waits for
      for (int j = max(0, it - kPairStages); ok && j < it; ++j)
        ok = mbar_wait(&sm.empty[j % kPairStages], (j / kPairStages) & 1, kStatusTimeoutMma, abort_flag, p.status);
    }
  } else if (warp == 1 && rank != 0) {
    // the leader issues the pair's MMAs
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    // The whole warp runs the loop and one lane issues, so that the descriptors stay in uniform registers.  (Inside a
    // branch of one lane every operand of every instruction is moved there first: 955 cycles a stage of nvfp4.)
    const uint64_t da = smem_desc_sw128(smem_u32(sm.a[0]), 16, 1024), db = smem_desc_sw128(smem_u32(sm.b[0]), 16, 1024);
    const uint64_t dsa = smem_desc_scales(smem_u32(sm.sa[0])), dsb = smem_desc_scales(smem_u32(sm.sb[0]));
    // s: the stage whose MMAs are next; (sn, phn): the stage whose scales are copied next, at most one ahead, into
    // buffer bufn, last read by the MMAs of stage s_old (kSfBufs before; with as many buffers as stages the ring itself
    // has waited for those)
    int s = 0, buf = 0, sn = 0, bufn = 0, s_old = 0;
    uint32_t phn = 0, ph_old = 0;
    const int my_tiles = cluster < p.num_tiles ? (p.num_tiles - 1 - cluster) / clusters + 1 : 0;
    int64_t left = (int64_t)my_tiles * p.ksteps;  // stages whose scales have not been copied
    int64_t copied = 0;
    int kn = 0;  // K step of stage sn
    auto copy_tile = [&](int j, int nt) {  // scale tile j along K of stage sn (the elected lane)
      const uint32_t sfa = tmem + kPairSfCol + bufn * kSfBufCols, sfb = sfa + 4 * kStageTiles;
      const uint64_t osa = (uint64_t)(sn * (kSaBytes >> 4)), osb = (uint64_t)(sn * (kSbBytes >> 4));
      if (j < nt) {
        tmem_cp_scales<2>(sfa + 4 * j, dsa + osa + j * (kFp4TileBytes >> 4));
        tmem_cp_scales<2>(sfb + 8 * j, dsb + osb + j * (kFp4TileBytes >> 4));
        tmem_cp_scales<2>(sfb + 8 * j + 4, dsb + osb + (kSaBytes >> 4) + j * (kFp4TileBytes >> 4));
      }
    };
    auto advance = [&] {  // stage sn's copies have been issued
      if (kSfBufs < kPairStages && copied >= kSfBufs)
        if (++s_old == kPairStages) s_old = 0, ph_old ^= 1;
      ++copied;
      --left;
      if (++sn == kPairStages) sn = 0, phn ^= 1;
      if (++bufn == kSfBufs) bufn = 0;
      if (++kn == p.ksteps) kn = 0;
    };
    int tl = 0;
    bool ok = true, ahead = false;  // ahead: the scales of stage s have been copied
    for (int t = cluster; ok && t < p.num_tiles; t += clusters, ++tl) {
      // both CTAs have read the columns shared with the previous tile's accumulator
      if (tl > 0) {
        ok = mbar_wait_cluster(&sm.acc_free, (tl - 1) & 1, kStatusTimeoutSoftmax, abort_flag, p.status);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
      }
      const uint32_t d = tmem + ((tl & 1) ? kPairAcc1 : 0);
      for (int k = 0; k < p.ksteps; ++k) {
        if (!ahead) {
          ok = mbar_wait_cluster(&sm.full[sn], phn, kStatusTimeoutTmaFull, abort_flag, p.status);
          if (kSfBufs < kPairStages && copied >= kSfBufs)
            ok = ok && mbar_wait(&sm.empty[s_old], ph_old, kStatusTimeoutMma, abort_flag, p.status);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          if constexpr (NV) {
            const int nt = min(kStageTiles, p.ktiles - kn * kStageTiles);
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < kStageTiles; ++j) copy_tile(j, nt);
            }
            __syncwarp();
            advance();
          }
        }
        // nvfp4: the next stage's scales go between this stage's MMAs if it has landed and its buffer is free (9472 x
        // 16384 x 5120: 317 us against 341 with all copies first).  mxfp4, with half as many, has them first, in one
        // go with its MMAs: 274 us there, 286 with the copies between, and 311 with no more than the votes and fences here.
        bool next = false;
        if constexpr (NV) {
          next = left > 0 && mbar_try_wait(smem_u32(&sm.full[sn]), phn);
          if (kSfBufs < kPairStages && copied >= kSfBufs) next = next && mbar_try_wait(smem_u32(&sm.empty[s_old]), ph_old);
          next = __all_sync(0xffffffffu, next);
          tc_fence_after();
        }
        const uint32_t sfa = tmem + kPairSfCol + buf * kSfBufCols, sfb = sfa + 4 * kStageTiles;
        const int nk = min(4, (p.K - k * kBK + 63) / 64), nt = !NV || next ? min(kStageTiles, p.ktiles - kn * kStageTiles) : 0;
        const uint64_t oa = (uint64_t)(s * (kABytes >> 4));
        if (elect_one()) {
          if constexpr (!NV) {
#pragma unroll
            for (int j = 0; j < kStageTiles; ++j) copy_tile(j, nt);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk < nk) {
              const int j = NV ? kk : kk >> 1;
              mma_fp4_ss<NV, 2>(d, da + oa + 2 * kk, db + oa + 2 * kk, idesc_fp4(NV, kPairBM, kBN, NV ? 0 : (kk & 1) * 2),
                                sfa + 4 * j, sfb + 8 * j, (k > 0 || kk > 0) ? 1u : 0u);
            }
            if (NV && kk < kStageTiles) copy_tile(kk, nt);
          }
          mma_commit_pair(&sm.empty[s]);
        }
        __syncwarp();
        if (!NV || next) advance();
        ahead = next;
        if (++s == kPairStages) s = 0;
        if (++buf == kSfBufs) buf = 0;
      }
      if (!ok) break;
      if (elect_one()) mma_commit_pair(&sm.acc_full[tl & 1]);
      __syncwarp();
    }
    if (elect_one()) {
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
      const bool any_far = NV && __any_sync(0xffffffffu, far_out(tra));
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
        if (any_far) {  // one vote a tile, so that the warp stays together (32760 x 8960 x 1536 nvfp4: 240 us, 247 by lane)
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float4 f = f4[q];
            const float a = __uint_as_float(v[2 * q]), b = __uint_as_float(v[2 * q + 1]);
            const bool far = far_out(tra);
            o[q] = pack_out<FP16>(far ? apply_factors_far(a, tra, f.x, f.y) : apply_factors(a, tra, f.x, f.y),
                                  far ? apply_factors_far(b, tra, f.z, f.w) : apply_factors(b, tra, f.z, f.w));
          }
        } else {
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float4 f = f4[q];
            o[q] = pack_out<FP16>(apply_factors(__uint_as_float(v[2 * q]), tra, f.x, f.y),
                                  apply_factors(__uint_as_float(v[2 * q + 1]), tra, f.z, f.w));
          }
        }
        if (p.rows16) {  // a box of 32 x 32 by TMA, 64-byte swizzle
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
  // The leader's last commit arrives in both CTAs, at some time after it is issued: neither leaves, or lets its shared
  // memory go, before its own barrier has been reached.  (The leader has waited; here the CTA's last tile is stored, so
  // the arrival is at most moments away.)
  if (rank != 0 && warp == 1) {
    if (elect_one()) mbar_wait(&sm.drain, 0, kStatusTimeoutMma, nullptr, p.status);
    __syncwarp();
  }
  cluster_sync();  // the pair's barriers and tensor memory are no longer in use by the other CTA
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------- few rows
// For few rows of x, D^T = B A^T: 128 rows of the weight B are the MMA's 128 rows and a tile of x's rows its N, so one
// token costs a tile of 32 columns, and the K loop of a tile is split over a cluster of up to six CTAs.  Each leaves
// its fp32 part in its shared memory, [column of x's tile][128 rows], and adds a share of the columns over all
// parts in rank order (the same sums every time), applies factors and bias and stores runs of the output row.
//   warp 0      producer (ring of four stages, three for more than 32 rows of x: what fits); with `early` the grid was
//               launched to overlap the quantiser of x: the weight's part of the first stages is loaded before waiting
//               for it
//   warp 1      TMEM owner, scale copies and MMAs; the scales of each stage have their own columns
//   warps 2..5  accumulator to shared memory; all warps add and store
// Two CTAs fit an SM (half the tensor memory each): a stage is some 12 instructions to the tensor core, which one warp
// issues slower than the SM could load the stage.  (One token, 15360 x 5120, in 240 CTAs: 15.5 us with room for one CTA an
// SM, 12.9 us for two.  plan_small() now makes 120 CTAs of it, one an SM, in 12.0 us.)
// Bound by the latency of a CTA's K steps (twenty for that token) and of the start; the weight's bytes take 6.8 us from HBM.
// A tile of x starts on a scale tile: in tensor memory the MMA's scales have to start on an even column (of 32 rows
// each), an odd one is a "misaligned address".
constexpr int kSmallThreads = 192, kSmallStages = 4;
constexpr int kSmallBN = 128, kSmallTmem = 256, kSmallSfCol = 128;  // scales behind the accumulator's 128 columns
static_assert(kSmallSfCol + kSmallStages * 8 * kMaxTiles <= kSmallTmem, "columns of the stages' scales");

struct SmallBars {
  float2 col[kBM];  // factor and bias of the tile's weight rows
  uint64_t full[kSmallStages], empty[kSmallStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct SmallParams {
  Params g;          // M rows of x, N rows of the weight
  int bn;            // rows of x of a tile: a multiple of 32 up to 128, and 128 where there are several tiles
  int stages, stage_bytes;
  int tiles_x;       // tiles along x
  int split, per_split;  // CTAs of a cluster, K steps of each
  int early;
};

template <bool NV>
__global__ void __launch_bounds__(kSmallThreads, 2)
fp4_gemm_small_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                      const __grid_constant__ SmallParams sp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ SmallBars sm;
  const Params& p = sp.g;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = warp_id(), lane = lane_id();
  constexpr int kStageTiles = NV ? 4 : 2;
  const int tile = blockIdx.x / sp.split, rank = blockIdx.x % sp.split;  // rank = rank in the cluster
  const int tw = tile / sp.tiles_x, tx = tile % sp.tiles_x;
  const int k0 = rank * sp.per_split, k1 = min(p.ksteps, k0 + sp.per_split), steps = max(0, k1 - k0);
  const int x0 = tx * sp.bn;
  constexpr int kSfCols = 8 * kStageTiles;  // columns of a stage's scales
  uint8_t *const sA = ring, *const sB = ring + kABytes, *const sSa = sB + sp.bn * 128, *const sSb = sSa + kSaBytes;

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
    tmem_alloc(&sm.tmem_base, kSmallTmem);
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
      auto bytes_of = [&](int i) { return (uint32_t)min(kStageTiles, p.ktiles - (k0 + i) * kStageTiles) * kFp4TileBytes; };
      auto load_w = [&](int i, int s) {
        const int kt = (k0 + i) * kStageTiles;
        uint8_t* at = ring + s * sp.stage_bytes;
        const uint32_t bytes = bytes_of(i);
        mbar_arrive_expect_tx(&sm.full[s], kABytes + sp.bn * 128 + 2 * bytes);
        tma_load_2d(at, &tm_w, &sm.full[s], (k0 + i) * 128, tw * kBM);
        bulk_load(at + (sSa - sA), p.sb + ((int64_t)tw * p.ktiles + kt) * kFp4TileBytes, bytes, &sm.full[s]);
      };
      auto load_x = [&](int i, int s) {
        const int kt = (k0 + i) * kStageTiles;
        uint8_t* at = ring + s * sp.stage_bytes;
        tma_load_2d(at + kABytes, &tm_x, &sm.full[s], (k0 + i) * 128, x0);
        bulk_load(at + (sSb - sA), p.sa + ((int64_t)tx * p.ktiles + kt) * kFp4TileBytes, bytes_of(i), &sm.full[s]);
      };
      const int first = min(steps, sp.stages);
      for (int i = 0; i < first; ++i) load_w(i, i);
      if (sp.early) wait_for_previous_grid();
      for (int i = 0; i < first; ++i) load_x(i, i);
      int i = first, s = 0;
      uint32_t ph = 0;
      for (; i < steps; ++i) {
        if (!mbar_wait(&sm.empty[s], ph, kStatusTimeoutEmpty, abort_flag, p.status)) break;
        load_w(i, s);
        load_x(i, s);
        if (++s == sp.stages) s = 0, ph ^= 1;
      }
      for (int j = max(0, i - sp.stages); j < i; ++j)  // all copies land before the ring is used for the sums
        mbar_wait(&sm.full[j % sp.stages], (j / sp.stages) & 1, kStatusTimeoutTmaFull, nullptr, p.status);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the loop and one lane issues: the descriptors stay in uniform registers.  (Inside a branch of
    // one lane every operand of every instruction is moved there first, some 200 cycles an MMA and 40 a copy.)
    const uint64_t da = smem_desc_sw128(smem_u32(ring), 16, 1024), db = smem_desc_sw128(smem_u32(ring) + kABytes, 16, 1024);
    const uint64_t dsa = smem_desc_scales(smem_u32(ring) + (uint32_t)(sSa - sA));
    const uint64_t dsb = smem_desc_scales(smem_u32(ring) + (uint32_t)(sSb - sA));
    bool ok = true;
    int s = 0;  // the step's stage
    uint32_t ph = 0;
    for (int i = 0; i < steps; ++i) {
      const int k = k0 + i;
      ok = mbar_wait(&sm.full[s], ph, kStatusTimeoutTmaFull, abort_flag, p.status);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint64_t off = (uint64_t)(s * sp.stage_bytes) >> 4;
      // (the stage's columns were last read by the MMAs for which the ring has waited)
      const uint32_t sfa = tmem + kSmallSfCol + s * kSfCols, sfb = sfa + 4 * kStageTiles;
      const int nt = min(kStageTiles, p.ktiles - k * kStageTiles), nk = min(4, (p.K - k * kBK + 63) / 64);
      if (elect_one()) {
#pragma unroll
        for (int j = 0; j < kStageTiles; ++j)
          if (j < nt) {
            tmem_cp_scales<1>(sfa + 4 * j, dsa + off + j * (kFp4TileBytes >> 4));
            tmem_cp_scales<1>(sfb + 4 * j, dsb + off + j * (kFp4TileBytes >> 4));
          }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (kk < nk) {
            const int j = NV ? kk : kk >> 1;
            mma_fp4_ss<NV, 1>(tmem, da + off + 2 * kk, db + off + 2 * kk, idesc_fp4(NV, kBM, sp.bn, NV ? 0 : (kk & 1) * 2),
                              sfa + 4 * j, sfb + 4 * j, (i > 0 || kk > 0) ? 1u : 0u);
          }
        mma_commit(&sm.empty[s]);
      }
      __syncwarp();
      if (++s == sp.stages) s = 0, ph ^= 1;
    }
    if (elect_one()) {
      if (!ok) *abort_flag = 1;
      mma_commit(&sm.acc_full);
      mbar_wait(&sm.acc_full, 0, kStatusTimeoutMma, nullptr, p.status);
    }
  }
  // the MMAs are done and every copy has landed: the ring becomes the part's fp32 sums
  if (warp >= 2) {  // factors and biases of the weight rows, read while the operands come in
    const int r = threadIdx.x - 64, n = min(tw * kBM + r, p.N - 1);
    sm.col[r] = make_float2(NV ? __ldg(p.rb + n) : 1.f, p.bias != nullptr ? load_bias(p, n) : 0.f);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  float* part = reinterpret_cast<float*>(ring);
  if (warp >= 2) {
    const int wq = warp & 3, row = wq * 32 + lane;
    const uint32_t acc = tmem + ((uint32_t)(wq * 32) << 16);
    auto put = [&](int c, const uint32_t (&r)[32]) {
#pragma unroll
      for (int q = 0; q < 32; ++q) part[(c + q) * kBM + row] = steps > 0 ? __uint_as_float(r[q]) : 0.f;
    };
    uint32_t r0[32], r1[32];
    int c = 0;
    for (; c + 64 <= sp.bn; c += 64) {
      tmem_ld32(acc + c, r0);
      tmem_ld32(acc + c + 32, r1);
      tmem_wait_ld();
      put(c, r0);
      put(c + 32, r1);
    }
    if (c < sp.bn) {
      tmem_ld32(acc + c, r0);
      tmem_wait_ld();
      put(c, r0);
    }
  }
  if (sp.early) wait_for_previous_grid();  // the row factors of x are read below
  tc_fence_before();
  __syncthreads();
  if (sp.split > 1) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kSmallTmem);
  }
  // this CTA's share of x's rows: a warp takes eight of them at a time (that many loads in flight), a lane four weight
  // rows of each
  const int per = (sp.bn + sp.split - 1) / sp.split, c_end = min(min(sp.bn, p.M - x0), (rank + 1) * per);
  constexpr int kWarps = kSmallThreads / 32, kRows = 8;
  const int n = tw * kBM + lane * 4;
  float2 cf[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) cf[q] = sm.col[lane * 4 + q];
  for (int c0 = rank * per + warp; c0 < c_end; c0 += kWarps * kRows) {
    float v[kRows][4];
#pragma unroll
    for (int u = 0; u < kRows; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[u][q] = 0.f;
    for (int r = 0; r < sp.split; ++r) {
      const uint32_t from = sp.split > 1 ? cluster_map(part + lane * 4, r) : smem_u32(part + lane * 4);
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int c = c0 + u * kWarps;
        if (c < c_end) {
          const float4 q = ld_cluster_float4(from + c * (kBM * 4));
          v[u][0] += q.x;
          v[u][1] += q.y;
          v[u][2] += q.z;
          v[u][3] += q.w;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int c = c0 + u * kWarps;
      if (c >= c_end || n >= p.N) continue;
      const float ra = NV ? p.ra[x0 + c] : 1.f;
      const bool far = NV && far_out(ra);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[u][q] = far ? apply_factors_far(v[u][q], ra, cf[q].x, cf[q].y) : apply_factors(v[u][q], ra, cf[q].x, cf[q].y);
      uint16_t* d = static_cast<uint16_t*>(p.d) + (int64_t)(x0 + c) * p.ldd + n;
      const uint32_t lo = p.out_fp16 ? pack_out<true>(v[u][0], v[u][1]) : pack_out<false>(v[u][0], v[u][1]);
      const uint32_t hi = p.out_fp16 ? pack_out<true>(v[u][2], v[u][3]) : pack_out<false>(v[u][2], v[u][3]);
      if (p.rows16) {
        *reinterpret_cast<uint2*>(d) = make_uint2(lo, hi);
      } else {
        d[0] = (uint16_t)lo;
        if (n + 1 < p.N) d[1] = (uint16_t)(lo >> 16);
        if (n + 2 < p.N) d[2] = (uint16_t)hi;
        if (n + 3 < p.N) d[3] = (uint16_t)(hi >> 16);
      }
    }
  }
  if (sp.split > 1) {
    __syncthreads();
    cluster_sync();  // the other CTAs have read this one's part
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

template <bool NV, bool FP16>
void launch_pair(const Fp4Matrix& a, const Fp4Matrix& b, Params& p, int device, cudaStream_t stream) {
  const int smem = (int)sizeof(PairSmem) + 1024;
  const CUtensorMap ma = code_map(a, kBM), mb = code_map(b, kBM), sa = scale_map(a), sb = scale_map(b);
  configure<fp4_gemm_pair_kernel<NV, FP16>>(smem, device);
  fp4_gemm_pair_kernel<NV, FP16><<<2 * std::min(p.num_tiles, sm_count(device) / 2), kPairThreads, smem, stream>>>(
      ma, mb, sa, sb, p.rows16 ? out_map(p) : ma, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

constexpr int kSmallSmem = 109 * 1024;  // dynamic shared memory of a CTA of the few-rows kernel: two fit an SM

// Tiles, stages and split of the few-rows kernel.
SmallParams plan_small(const Params& p, int sms, bool early) {
  SmallParams sp;
  sp.g = p;
  sp.tiles_x = (p.M + kSmallBN - 1) / kSmallBN;
  sp.bn = sp.tiles_x > 1 ? kSmallBN : (p.M + 31) / 32 * 32;
  sp.stage_bytes = kABytes + sp.bn * 128 + 2 * kSaBytes;
  sp.stages = std::min(kSmallStages, (kSmallSmem - 1024) / sp.stage_bytes);
  // CTAs for up to four fifths of the places (two an SM; 236 of 148 SMs): above that, and with clusters of more than six,
  // they no longer all run at once (16 x 5120 x 5120 nvfp4: 10.0 us with 160 to 240 CTAs, 15.1 us with 280)
  const int tiles = ((p.N + kBM - 1) / kBM) * sp.tiles_x;
  sp.split = std::max(1, std::min({6, sms * 2 * 4 / 5 / std::max(tiles, 1), p.ksteps}));
  sp.per_split = (p.ksteps + sp.split - 1) / sp.split;
  sp.early = early ? 1 : 0;
  return sp;
}

// Which kernel: up to 128 rows of x the few-rows kernel reads the weight once and wastes no half of a 256-row tile; above
// it stays ahead while its 128 x 128 tiles do not fill the GPU (256 x 5120 x 15360: 20.4 us against 27.3; 1024 x 1536 x
// 1536: 10.2 against 11.1) and falls behind when they do (512 x 5120 x 5120: 20.1 against 18.6).
bool few_rows(const Params& p, int sms) {
  if (p.M <= kSmallBN) return true;
  const int64_t tiles = (int64_t)((p.N + kBM - 1) / kBM) * ((p.M + kSmallBN - 1) / kSmallBN);
  return tiles <= sms * 7 / 8;
}

template <bool NV>
void launch_small(const Fp4Matrix& a, const Fp4Matrix& b, const SmallParams& sp, int device, cudaStream_t stream) {
  const int tiles = ((sp.g.N + kBM - 1) / kBM) * sp.tiles_x;
  const CUtensorMap mw = code_map(b, kBM), mx = code_map(a, sp.bn);
  // the ring, and the fp32 sums that take its place
  const int smem = std::max(sp.stages * sp.stage_bytes, sp.bn * kBM * 4) + 1024;
  configure<fp4_gemm_small_kernel<NV>>(kSmallSmem, device);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * sp.split));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)sp.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = sp.early ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fp4_gemm_small_kernel<NV>, mw, mx, sp));
}

// early: the kernel before this one on the stream is the quantiser that wrote a, launched without overlap itself.
template <bool NV>
void launch(const Fp4Matrix& a, const Fp4Matrix& b, Params& p, int device, cudaStream_t stream, bool early) {
  const int sms = sm_count(device);
  if (few_rows(p, sms)) launch_small<NV>(a, b, plan_small(p, sms, early), device, stream);
  else if (p.out_fp16) launch_pair<NV, true>(a, b, p, device, stream);
  else launch_pair<NV, false>(a, b, p, device, stream);
}

// d [a.rows, b.rows] (bf16 or fp16, contiguous) = a b^T + bias, on the current device and stream.
void gemm(const Fp4Matrix& a, const Fp4Matrix& b, const c10::optional<at::Tensor>& bias, at::Tensor& d,
          cudaStream_t stream, bool early) {
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
  p.rows16 = (reinterpret_cast<uintptr_t>(p.d) | (uintptr_t)(2 * N)) % 16 == 0;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.ktiles = (int)a.ktiles();
  p.ksteps = (int)((K + kBK - 1) / kBK);
  p.tiles_m = (int)((M + kPairBM - 1) / kPairBM);
  p.tiles_n = (int)((N + kBN - 1) / kBN);
  DMAD_VALUE_CHECK((int64_t)p.tiles_m * p.tiles_n <= INT32_MAX, "fp4_linear: too many output tiles");
  p.num_tiles = p.tiles_m * p.tiles_n;
  const int device = d.get_device();
  p.status = device_status_ptr(device);
  a.nv ? launch<true>(a, b, p, device, stream, early) : launch<false>(a, b, p, device, stream, early);
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
  gemm(q, w, b, y, stream, true);
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
  gemm(q, w, b, y, at::cuda::getCurrentCUDAStream(), false);
  return y;
}

}  // namespace dmad
