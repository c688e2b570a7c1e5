// A persistent tcgen05 GEMM on pairs of CTAs, for 8-bit integers and for 16-bit floating point, with the epilogue as a
// parameter.
//
//   acc[m, n] = sum_k A[m, k] B[n, k]        (int32 or fp32, in tensor memory)
//
// A pair of CTAs works on each 256 x 256 tile (cta_group::2), one CTA an SM: each CTA holds 128 rows of A and of the
// accumulator and loads 128 of B's 256 rows, so that a stage of 128 bytes of K moves 32 KB into an SM in the 512 cycles of
// its MMAs (a 128 x 256 tile of one CTA: 48 KB, more than an SM gets from the L2 in that time).
//   warp 0      producer of its own CTA's operands, which complete on the leader's barriers
//   warp 1      leader CTA: issues the MMAs.  The whole warp runs the loop and one lane issues, so that the descriptors stay
//               in uniform registers
//   warps 2..   epilogue of the CTA's 128 rows: two or four warps a lane quarter, every second or fourth 32 columns each
// The two accumulators take the 512 columns of tensor memory, so that a tile's epilogue runs beside the next one's MMAs.
// An operand is read K-major ([rows, K]) or, 16-bit types, MN-major ([K, rows]) where it lies.
// Tiles that would leave half of the pairs or more without work (all of them, where they are few; those of the last round
// else) have their K steps spread over several pairs: these store the accumulators as they are, 256 x 256 numbers an item, and
// a second kernel adds a tile's parts in order and does what the epilogue does.  (tile_split() says when.)
// Every mbarrier wait is bounded (2 s), records a status code and makes all roles leave.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <c10/cuda/CUDAException.h>
#include <torch/extension.h>
#include "checks.h"
#include "common.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace dmad {

int* device_status_ptr(int device);

enum class Mma { kI8, kBf16, kF16 };

// Instruction descriptor (bits as for bf16): signed 8-bit integers (code 1) into s32 (code 2), bf16 (1) or fp16 (0) into
// f32 (1).
__host__ __device__ constexpr uint32_t idesc_of(Mma kind, int M, int N, bool a_mn, bool b_mn) {
  const uint32_t ab = kind == Mma::kF16 ? 0u : 1u;
  return ((kind == Mma::kI8 ? 2u : 1u) << 4) | (ab << 7) | (ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// D[tmem] (+)= A[smem] B[smem]^T over 32 bytes of K.  CG = 2: for a CTA pair, A's and D's rows split over the two and B's
// rows loaded half by each.
template <Mma KIND, int CG>
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
#define DMAD_MMA(GROUP, TYPE)                                                                                             \
  asm volatile("{\n\t.reg .pred p;\n\t"                                                                                  \
               "setp.ne.b32 p, %4, 0;\n\t"                                                                               \
               "tcgen05.mma.cta_group::" GROUP ".kind::" TYPE " [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc),   \
               "l"(b_desc), "r"(idesc), "r"(accumulate)                                                                  \
               : "memory")
  static_assert(CG == 2 || KIND == Mma::kI8, "one CTA's MMAs: 8-bit integers (the few-rows product)");
  if constexpr (CG == 1) DMAD_MMA("1", "i8");
  else if constexpr (KIND == Mma::kI8) DMAD_MMA("2", "i8");
  else DMAD_MMA("2", "f16");
#undef DMAD_MMA
}

constexpr int kPairM = 256, kPairN = 256, kPairHalf = 128;
constexpr int kPairTileBytes = kPairHalf * 128;  // an operand's rows of a stage in one CTA: 16 KB

struct PairGemm {
  int M, N;
  int ksteps;             // stages along K: 128 bytes each
  int k_last;             // MMAs (32 bytes) of the last stage
  int tiles_m, tiles_n, items;  // work items: `whole` tiles, then `split` of each other tile
  int whole, split, per_split;  // per_split: K steps of a part
  int a_mn, b_mn;         // 1: stored [K, rows]
  int b_old;              // (early 1) B is older than the kernel before: its first stages are loaded before the wait
  int early;              // launched to overlap the kernel before it: 1 reads what that writes, 2 does not (operands and
                          // epilogue's inputs older); either way results are stored after its end
  int* status;

  __device__ __forceinline__ void tile(int item, int& tm, int& tn) const {
    // column-major raster within groups of 8 M-tiles: neighbouring pairs share B tiles in L2
    constexpr int kGroup = 8;
    const int t = item < whole ? item : whole + (item - whole) / split, group = t / (kGroup * tiles_n), first = group * kGroup;
    const int gm = min(kGroup, tiles_m - first), in = t % (kGroup * tiles_n);
    tm = first + in % gm;
    tn = in / gm;
  }
  __device__ __forceinline__ void steps(int item, int& k0, int& k1) const {
    k0 = item < whole ? 0 : (item - whole) % split * per_split;
    k1 = item < whole ? ksteps : min(ksteps, k0 + per_split);
  }
  __host__ __device__ __forceinline__ int split_tiles() const { return (items - whole) / split; }
};

// What an epilogue warp knows of its place.
struct EpiPlace {
  uint8_t* stage;   // the warp's shared memory
  float2* col;      // [2][256], shared by the epilogue warps
  int wq, group, lane, thread;  // lane quarter; the warp's chunks of 32 columns: group, group + kWarps / 4, ..
  uint32_t rank;
};

template <int STAGES, int WARPS, int OUT_BYTES, bool SHARED>
struct PairGemmSmem {
  uint8_t a[STAGES][kPairTileBytes];
  uint8_t b[STAGES][kPairTileBytes];
  uint8_t out[WARPS][OUT_BYTES];
  float2 col[2][SHARED ? kPairN : 1];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t acc_full[2], acc_free[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};

// One operand's 128 rows from r0 of K step k.  MN-major: two boxes of 64 rows, [64 of K][64 rows] each.
__device__ __forceinline__ void load_pair_operand(uint8_t* dst, const CUtensorMap* tm, uint32_t bar, int k, int r0, int step,
                                                  bool mn) {
  if (!mn) {
    tma_load_2d_pair(dst, tm, bar, k * step, r0);
  } else {
    tma_load_2d_pair(dst, tm, bar, r0, k * step);
    tma_load_2d_pair(dst + 8192, tm, bar, r0 + 64, k * step);
  }
}

// Epi: kStages, kWarps (8 or 16), kOutBytes (shared memory of a warp), kShared (the column factors are used: the epilogue's
// warps, eight of them, meet once a tile), kAhead (a chunk is read from tensor memory while the one before is worked on; short
// epilogues), Args (passed to the kernel), and
//   Epi(args, gemm, place)
//   first(item)                 before the first tile
//   begin(item, next, parity)   before the tile's accumulator is waited for; next: the item after it, or -1
//   met(next)                   behind the warps' barrier (kShared only)
//   chunk(c, v)                 the accumulator's columns 32 c .. 32 c + 31 of the lane's row
// (of a part only the calls that the barrier's warps share are made)
// Columns 32 c .. of the lane's row of a part, through 2 KB of shared memory: twice 16 columns of 32 rows (64-byte swizzle).
__device__ __forceinline__ void store_part(const CUtensorMap* map, const EpiPlace& at, int part, int c, const uint32_t (&v)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (at.lane == 0) tma_store_wait_read();
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4*>(at.stage + at.lane * 64 + ((q ^ ((at.lane >> 1) & 3)) << 4)) =
          make_uint4(v[16 * h + 4 * q], v[16 * h + 4 * q + 1], v[16 * h + 4 * q + 2], v[16 * h + 4 * q + 3]);
    fence_proxy_async_smem();
    __syncwarp();
    if (at.lane == 0) tma_store_2d(map, at.stage, c * 32 + h * 16, part * kPairM + (int)at.rank * kPairHalf + at.wq * 32);
  }
}

template <Mma KIND, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * Epi::kWarps, 1)
pair_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_parts, const __grid_constant__ typename Epi::Args args,
                 const PairGemm p) {
  constexpr int kStages = Epi::kStages, kWarps = Epi::kWarps, kGroups = kWarps / 4, kChunks = kPairN / 32 / kGroups;
  static_assert(!Epi::kShared || 32 * kWarps == kPairN, "a column a thread");
  using Smem = PairGemmSmem<kStages, kWarps, Epi::kOutBytes, Epi::kShared>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = &sm.abort_flag;
  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  constexpr int kStep = KIND == Mma::kI8 ? 128 : 64;  // elements of K of a stage

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);  // the leader's counts both CTAs' bytes; the other CTA's is not used
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_free[b], 2 * kWarps);
    }
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
  }
  launch_dependents();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  if (p.early != 0 && warp > 1) wait_for_previous_grid();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int it = 0, s = 0, b_loaded = 0;  // stages whose part of B has been loaded
      uint32_t ph = 0;
      bool ok = true;
      if (p.early == 1 && p.b_old && pair < p.items) {
        int tm, tn, k0, k1;
        p.tile(pair, tm, tn);
        p.steps(pair, k0, k1);
        b_loaded = min(kStages, k1 - k0);
        for (int j = 0; j < b_loaded; ++j) {
          if (rank == 0) mbar_arrive_expect_tx(&sm.full[j], 4 * kPairTileBytes);
          load_pair_operand(sm.b[j], &tm_b, cluster_map(&sm.full[j], 0), k0 + j, tn * kPairN + (int)rank * kPairHalf, kStep, p.b_mn);
        }
      }
      if (p.early == 1) wait_for_previous_grid();
      for (int t = pair; ok && t < p.items; t += pairs) {
        int tm, tn, k0, k1;
        p.tile(t, tm, tn);
        p.steps(t, k0, k1);
        const int ra = tm * kPairM + (int)rank * kPairHalf, rb = tn * kPairN + (int)rank * kPairHalf;
        for (int k = k0; k < k1; ++k, ++it) {
          if (!(ok = mbar_wait(&sm.empty[s], ph ^ 1, kStatusTimeoutEmpty, abort_flag, p.status))) break;
          // boxes are written, and counted, whole: zeros past the operands
          const uint32_t full = cluster_map(&sm.full[s], 0);
          if (it >= b_loaded) {
            if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], 4 * kPairTileBytes);
            load_pair_operand(sm.b[s], &tm_b, full, k, rb, kStep, p.b_mn);
          }
          load_pair_operand(sm.a[s], &tm_a, full, k, ra, kStep, p.a_mn);
          if (++s == kStages) s = 0, ph ^= 1;
        }
      }
      // all issued copies land before a CTA's shared memory goes away
      if (rank == 0)
        for (int j = max(0, it - kStages); j < it; ++j)
          mbar_wait_cluster(&sm.full[j % kStages], (j / kStages) & 1, kStatusTimeoutTmaFull, nullptr, p.status);
      // and so do the leader's arrivals for the last stages, which nobody else waits for
      for (int j = max(0, it - kStages); ok && j < it; ++j)
        ok = mbar_wait(&sm.empty[j % kStages], (j / kStages) & 1, kStatusTimeoutMma, abort_flag, p.status);
    }
  } else if (warp == 1 && rank != 0) {
    // the leader issues the pair's MMAs
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    // 32 bytes of K further: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
    const uint64_t da = p.a_mn ? smem_desc_sw128(smem_u32(sm.a[0]), 8192, 1024) : smem_desc_sw128(smem_u32(sm.a[0]), 16, 1024);
    const uint64_t db = p.b_mn ? smem_desc_sw128(smem_u32(sm.b[0]), 8192, 1024) : smem_desc_sw128(smem_u32(sm.b[0]), 16, 1024);
    const uint64_t ka = p.a_mn ? 2048 >> 4 : 32 >> 4, kb = p.b_mn ? 2048 >> 4 : 32 >> 4;
    const uint32_t idesc = idesc_of(KIND, kPairM, kPairN, p.a_mn != 0, p.b_mn != 0);
    int s = 0, tl = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = pair; ok && t < p.items; t += pairs, ++tl) {
      if (tl >= 2) {  // both CTAs have read this accumulator
        ok = mbar_wait_cluster(&sm.acc_free[tl & 1], ((tl >> 1) - 1) & 1, kStatusTimeoutSoftmax, abort_flag, p.status);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
      }
      const uint32_t d = tmem + (tl & 1) * kPairN;
      int k0, k1;
      p.steps(t, k0, k1);
      for (int k = k0; k < k1; ++k) {
        ok = mbar_wait_cluster(&sm.full[s], ph, kStatusTimeoutTmaFull, abort_flag, p.status);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        const uint64_t off = (uint64_t)(s * (kPairTileBytes >> 4));
        const int nk = k == p.ksteps - 1 ? p.k_last : 4;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < nk) mma_ss<KIND, 2>(d, da + off + kk * ka, db + off + kk * kb, idesc, (k > k0 || kk > 0) ? 1u : 0u);
          mma_commit_pair(&sm.empty[s]);
        }
        __syncwarp();
        if (++s == kStages) s = 0, ph ^= 1;
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
    // ------------------------------------------------------------ epilogue (warps 2..)
    const int ew = warp - 2;
    const EpiPlace place{sm.out[ew], &sm.col[0][0], warp & 3, ew >> 2, lane, (int)threadIdx.x - 64, rank};
    const uint32_t lane_base = (uint32_t)(place.wq * 32) << 16;
    Epi epi(args, p, place);
    if (pair < p.items) epi.first(pair);
    int tl = 0;
    for (int t = pair; t < p.items; t += pairs, ++tl) {
      const int next = t + pairs < p.items ? t + pairs : -1;
      const bool part = t >= p.whole;
      if (Epi::kShared || !part) epi.begin(t, next, tl & 1);
      bool ok = mbar_wait(&sm.acc_full[tl & 1], (tl >> 1) & 1, kStatusTimeoutMma, abort_flag, p.status);
      if constexpr (Epi::kShared) {  // all warps leave together, since the barrier counts them
        if (named_bar_any(1, 32 * kWarps, !ok)) break;
        epi.met(next);
      } else {
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + lane_base + (tl & 1) * kPairN;
      const uint32_t freed = cluster_map(&sm.acc_free[tl & 1], 0);
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(freed);
      };
      auto finish = [&](int c, const uint32_t (&v)[32]) {
        if (part) store_part(&tm_parts, place, t - p.whole, c, v);
        else epi.chunk(c, v);
      };
      if constexpr (Epi::kAhead) {
        uint32_t r[2][32];
        tmem_ld32(acc + place.group * 32, r[0]);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          tmem_wait_ld();
          if (i + 1 < kChunks) tmem_ld32(acc + (kGroups * (i + 1) + place.group) * 32, r[(i + 1) & 1]);
          else release();
          finish(kGroups * i + place.group, r[i & 1]);
        }
      } else {
#pragma unroll 1
        for (int c = place.group; c < kPairN / 32; c += kGroups) {
          uint32_t r[32];
          tmem_ld32(acc + c * 32, r);
          tmem_wait_ld();
          if (c + kGroups >= kPairN / 32) release();
          finish(c, r);
        }
      }
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

// ---------------------------------------------------------------- rows of 16-bit results
template <bool FP16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (FP16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}

// A 16-bit matrix [M, N] that leaves in boxes of 32 x 32: by TMA (64-byte swizzle) where its rows start on 16 bytes, else
// through shared memory in runs of 32 bytes.
struct OutRows {
  uint16_t* d;
  int64_t ld;
  int M, N;
  bool tma;
};

// Columns nc .. nc + 31 of the warp's rows m0 .. m0 + 31 (o: the lane's row), through 2 KB of shared memory.
__device__ __forceinline__ void store_rows(const OutRows& out, const CUtensorMap* map, uint8_t* stage, int m0, int nc,
                                           const uint32_t (&o)[16]) {
  const int lane = lane_id();
  if (nc >= out.N || m0 >= out.M) return;
  if (out.tma) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) tma_store_2d(map, stage, nc, m0);
  } else {
    uint16_t(*t)[18] = reinterpret_cast<uint16_t(*)[18]>(stage);
    uint16_t* d0 = out.d + (int64_t)m0 * out.ld + nc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 8; ++q) *reinterpret_cast<uint32_t*>(&t[lane][2 * q]) = o[8 * h + q];
      __syncwarp();
      const int cc = lane & 15, n = 16 * h + cc;
      for (int r = lane >> 4; r < 32; r += 2)
        if (m0 + r < out.M && nc + n < out.N) d0[(int64_t)r * out.ld + n] = t[r][cc];
    }
  }
}

// Row m and first column n of a thread of such a kernel, and where the first part's four numbers are; false past the matrix.
__device__ __forceinline__ bool part_place(const PairGemm& p, int& m, int& n, int64_t& at) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), col = (threadIdx.x & 63) * 4;
  int tm, tn;
  p.tile(p.whole + blockIdx.y * p.split, tm, tn);
  m = tm * kPairM + row;
  n = tn * kPairN + col;
  at = ((int64_t)blockIdx.y * p.split * kPairM + row) * kPairN + col;
  return m < p.M && n < p.N;
}
constexpr int64_t kPartStep = (int64_t)kPairM * kPairN;  // from one part to the next

// Four columns from n of row m of a 16-bit matrix.
template <bool FP16>
__device__ __forceinline__ void store4(const OutRows& o, int m, int n, const float (&v)[4]) {
  uint16_t* d = o.d + (int64_t)m * o.ld + n;
  const uint32_t lo = pack16<FP16>(v[0], v[1]), hi = pack16<FP16>(v[2], v[3]);
  if (o.tma && n + 4 <= o.N) {
    *reinterpret_cast<uint2*>(d) = make_uint2(lo, hi);
  } else {
    d[0] = (uint16_t)lo;
    if (n + 1 < o.N) d[1] = (uint16_t)(lo >> 16);
    if (n + 2 < o.N) d[2] = (uint16_t)hi;
    if (n + 3 < o.N) d[3] = (uint16_t)(hi >> 16);
  }
}

// A row of numbers of any of three types: 0 fp32, 1 bf16, 2 fp16; none: zeros.
struct FloatRow {
  const void* p;
  int type;
  __device__ __forceinline__ float at(int n) const {
    if (p == nullptr) return 0.f;
    if (type == 0) return __ldg(static_cast<const float*>(p) + n);
    if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[n]);
    return __half2float(static_cast<const __half*>(p)[n]);
  }
};

// ---------------------------------------------------------------- host
inline FloatRow float_row(const c10::optional<at::Tensor>& t) {
  if (!(t.has_value() && t->defined())) return FloatRow{nullptr, 0};
  return FloatRow{t->data_ptr(), t->scalar_type() == at::kFloat ? 0 : t->scalar_type() == at::kBFloat16 ? 1 : 2};
}

// The bias [N] of a linear layer, contiguous; a ValueError where it does not fit.
inline c10::optional<at::Tensor> checked_bias(const c10::optional<at::Tensor>& bias, int64_t N, const at::Device& device,
                                              const char* name) {
  if (!(bias.has_value() && bias->defined())) return c10::nullopt;
  DMAD_VALUE_CHECK(bias->device() == device && bias->dim() == 1 && bias->size(0) == N && is_float_type(bias->scalar_type()),
                   std::string(name) + ": bias must be bf16, fp16 or fp32 (" + num(N) + ",) on the device of w, got " +
                       dtype_name(bias->scalar_type()) + " " + shape_text(*bias));
  return bias->contiguous();
}

inline CUtensorMap out_rows_map(const OutRows& o) {  // 16-bit elements, whichever
  const uint64_t dims[2] = {(uint64_t)o.N, (uint64_t)o.M};
  const uint64_t strides[1] = {(uint64_t)o.ld * 2};
  const uint32_t box[2] = {32u, 32u};
  return make_tmap_bf16(o.d, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

// TMA writes whole pieces of 16 bytes, so the columns that it may write have to end on one: where N does not (one half of a
// row beside the other), runs of 32 bytes are stored instead.
inline OutRows out_rows(void* d, int64_t ld, int64_t M, int64_t N) {
  return OutRows{static_cast<uint16_t*>(d), ld, (int)M, (int)N,
                 (reinterpret_cast<uintptr_t>(d) | (uintptr_t)(2 * ld) | (uintptr_t)(2 * N)) % 16 == 0};
}

// An operand's map: rows x 128 bytes of a K-major matrix, or 64 x 64 of an MN-major one.
inline CUtensorMap operand_map(const void* base, int64_t rows, int64_t K, int64_t ld, int bytes, bool mn) {
  const uint64_t dims[2] = {(uint64_t)(mn ? rows : K), (uint64_t)(mn ? K : rows)};
  const uint64_t strides[1] = {(uint64_t)(ld * bytes)};
  const uint32_t box[2] = {(uint32_t)(128 / bytes), mn ? 64u : (uint32_t)kPairHalf};
  return bytes == 1 ? make_tmap_u8(base, 2, dims, strides, box) : make_tmap_bf16(base, 2, dims, strides, box);
}

// Parts of each tile of a round that fills no more than half of the pairs: as many as fill them, of four stages on average at
// least (all of one length but the last part, which may be shorter).  After whole rounds only where that saves twelve stages
// (some 3 us), for which the parts' kernel is paid.
inline int tile_split(int64_t tiles, int64_t stages, int pairs, bool only) {
  if (tiles == 0 || 2 * tiles > pairs) return 1;
  const int64_t split = std::max<int64_t>(1, std::min(pairs / tiles, stages / 4));
  return only || stages - stages / split >= 12 ? (int)split : 1;
}

inline PairGemm pair_gemm(int64_t M, int64_t N, int64_t K, int bytes, bool a_mn, bool b_mn, int device) {
  PairGemm p;
  const int64_t step = 128 / bytes, per_mma = 32 / bytes;
  p.M = (int)M;
  p.N = (int)N;
  p.ksteps = (int)((K + step - 1) / step);
  p.k_last = (int)((K - (int64_t)(p.ksteps - 1) * step + per_mma - 1) / per_mma);
  p.tiles_m = (int)((M + kPairM - 1) / kPairM);
  p.tiles_n = (int)((N + kPairN - 1) / kPairN);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  DMAD_VALUE_CHECK(tiles <= INT32_MAX / 4, "too many output tiles");
  const int pairs = sm_count(device) / 2;
  p.whole = (int)(tiles / pairs * pairs);
  const int split = tile_split(tiles - p.whole, p.ksteps, pairs, p.whole == 0);
  p.per_split = (p.ksteps + split - 1) / split;
  p.split = (p.ksteps + p.per_split - 1) / p.per_split;  // every part has a step
  if (p.split == 1) p.whole = (int)tiles;
  p.items = p.whole + (int)(tiles - p.whole) * p.split;
  p.a_mn = a_mn ? 1 : 0;
  p.b_mn = b_mn ? 1 : 0;
  p.early = p.b_old = 0;
  p.status = device_status_ptr(device);
  return p;
}

// Raises a kernel's dynamic shared memory limit, once a device.
template <auto Kernel>
void raise_smem(int smem, int device) {
  static std::array<std::atomic<bool>, 64> done{};
  if (device < 64 && done[device].load(std::memory_order_acquire)) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (device < 64) done[device].store(true, std::memory_order_release);
}

// Launch of a kernel that may overlap the end of the one before it (and then waits for it by itself).
template <class... Params, class... Args>
void launch_overlapping(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool early,
                        const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// Memory for the parts of p's divided tiles (undefined where there are none): [items, 256, 256] 32-bit numbers.
inline at::Tensor part_memory(const PairGemm& p, const at::TensorOptions& options) {
  if (p.split == 1) return at::Tensor();
  return at::empty({(int64_t)(p.items - p.whole) * kPairM, kPairN}, options.dtype(at::kInt).requires_grad(false));
}

template <Mma KIND, class Epi>
void launch_pair_gemm(const CUtensorMap& a, const CUtensorMap& b, const at::Tensor& parts, const typename Epi::Args& args,
                      const PairGemm& p, int device, cudaStream_t stream) {
  constexpr int smem = (int)sizeof(PairGemmSmem<Epi::kStages, Epi::kWarps, Epi::kOutBytes, Epi::kShared>) + 1024;
  static_assert(smem <= 232448 && Epi::kOutBytes >= 2048, "shared memory of an SM, of a part's rows");
  CUtensorMap mp = a;
  if (parts.defined()) {
    const uint64_t dims[2] = {(uint64_t)kPairN, (uint64_t)parts.size(0)};
    const uint64_t strides[1] = {(uint64_t)kPairN * 4};
    const uint32_t box[2] = {16u, 32u};
    mp = make_tmap(CU_TENSOR_MAP_DATA_TYPE_INT32, parts.data_ptr(), 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
  }
  raise_smem<pair_gemm_kernel<KIND, Epi>>(smem, device);
  launch_overlapping(pair_gemm_kernel<KIND, Epi>, dim3(2 * std::min(p.items, sm_count(device) / 2)), dim3(64 + 32 * Epi::kWarps), smem,
                     stream, p.early != 0, a, b, mp, args, p);
}

// Blocks of a kernel that adds parts, four columns a thread: four rows of a tile each.
inline dim3 part_grid(const PairGemm& p) { return dim3(kPairM / 4, (unsigned)p.split_tiles()); }
constexpr int kPartThreads = 256;

}  // namespace dmad
