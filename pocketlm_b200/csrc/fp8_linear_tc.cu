// The block-scaled FP8 linear for batches whose rows are e4m3 too:
//   out[t, n] = sum_g sx[t, g] sw[n / 128, g] sum_{k in group g} x[t, k] w[n, k],
// groups of 128 columns, 128 x 128 weight blocks.  A group's products are summed
// by tcgen05.mma kind::f8f6f4 (four steps of K = 32, exact products, fp32
// sums in tensor memory); its sum leaves tensor memory once and is added, times
// the group's scales, to an fp32 sum in registers.  One rounding to the
// output's type.  A 128-column group of e4m3 is one row of the 128B swizzle,
// so a pipeline stage is one group of both operands, loaded by TMA as stored;
// absent rows and columns arrive as zeros.
//
// Few rows (linear_rows_kernel).  The weight's rows
// are M (128 of them per CTA), the tokens N (16 to 128), so no tensor work is
// spent on absent tokens; the groups are cut over the CTAs of a cluster, whose
// sums are added through distributed shared memory in rank order (the same
// result on every run).  Measured at 1965 MHz: 64 x 24576 x 1536 13.4 us with the
// weight from memory (41 MB, 3.1 TB/s), 11.5 from L2; 1 x 2112 x 7168 8.6 and 6.8 us.
// Latency bounds it: the launch, the first bytes and the cluster's sum, then some
// 0.6 us per group and CTA, from the load over the products to the sums, whether
// the weight is in L2 or not.
//
// Many rows (linear_tiles_kernel).  256 tokens x up
// to 256 outputs per pair of CTAs and tile, two accumulators so that the sums
// of one group are read while the next is computed; persistent.  Measured:
// 4000 x 7168 x 16384 541 us in a loop of a second (1.74 PFLOP/s at the 1530 MHz
// that the power limit leaves), 476 us after a rest.  A group of a 256 x 256 tile
// takes 870 cycles, 520 of them products.  No unit is busy all the time (2000 x
// 7168 x 7168: tensor cores 51 % of the cycles, tensor memory 47 %, issue slots
// 51 %): the handing of two accumulators to and fro between products and sums,
// and the power, bound it.
#include <algorithm>

#include "fp8_gemv.cuh"
#include "router.cuh"
#include "rows.cuh"
#include "serving.cuh"
#include "tcgen05.cuh"

namespace moe {
namespace {

constexpr int kGroup = 128;  // columns per scale group: a stage of the pipeline

MOE_D bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xFFFFFFFFu, wait_or_abort(bar, parity, abort, kLinearWaitError));
}

// ------------------------------------------------------------------ few rows

constexpr int kRowsThreads = 192;  // warps 0-3: sums (a thread per weight row); 4: TMA; 5: products
constexpr int kWTileBytes = 128 * kGroup;
constexpr int kSumStride = 132;  // floats per token of a CTA's sums in shared memory: no bank is hit twice
template <int NT>
struct RowsShape {
  static constexpr int kStages = NT <= 32 ? 5 : NT <= 64 ? 4 : 6;
  static constexpr int kPerSm = NT <= 64 ? 2 : 1;  // CTAs that fit an SM
  static constexpr int kBufs = 4;                  // accumulators in tensor memory
  static constexpr int kCols = NT * kBufs < 32 ? 32 : NT * kBufs;
  static constexpr int kStageBytes = kWTileBytes + NT * kGroup;
  static constexpr int kPipeBytes = kStages * kStageBytes;
  static_assert(NT * kSumStride * 4 <= kPipeBytes, "the sums take the pipeline's place");
};
template <int NT>
struct RowsBarriers {
  uint64_t full[RowsShape<NT>::kStages], empty[RowsShape<NT>::kStages];
  uint64_t sum_full[RowsShape<NT>::kBufs], sum_empty[RowsShape<NT>::kBufs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

template <int NT>
size_t rows_smem(int groups) {
  return 1024 + RowsShape<NT>::kPipeBytes + sizeof(float) * NT * groups + sizeof(RowsBarriers<NT>);
}

// Four bytes into shared memory, on their way until copies4_wait().
MOE_D void copy4_async(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
MOE_D void copies4_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

MOE_D float4 ld_cluster(const float* p, uint32_t rank) {
  const uint32_t at = cluster_addr(p, rank);
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

// grid: (tile of 128 weight rows x cluster, tile of NT tokens); rank r of a
// cluster of S takes groups [r G / S, (r + 1) G / S).
template <typename O, int NT>
__global__ void __launch_bounds__(kRowsThreads) linear_rows_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                   const __grid_constant__ CUtensorMap map_w, LinearArgs a,
                                                                   int splits, int max_groups) {
  using Shape = RowsShape<NT>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale = reinterpret_cast<float*>(smem + Shape::kPipeBytes);  // [group][token]
  auto* bars = reinterpret_cast<RowsBarriers<NT>*>(scale + NT * max_groups);
  const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xFFFFFFFFu, tid / kWarp, 0);
  volatile int* abort = &bars->abort;
  const int rank = splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int tile = blockIdx.x / splits, n0 = tile * 128, t0 = blockIdx.y * NT;
  const int groups_all = static_cast<int>((a.cols + kGroup - 1) / kGroup);
  const int g0 = static_cast<int>(static_cast<int64_t>(rank) * groups_all / splits);
  const int groups = static_cast<int>(static_cast<int64_t>(rank + 1) * groups_all / splits) - g0;

  if (tid == 0) {
    for (int s = 0; s < Shape::kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < Shape::kBufs; ++b) {
      mbar_init(&bars->sum_full[b], 1);
      mbar_init(&bars->sum_empty[b], 4);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&bars->tmem_base, Shape::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // by 16 tokens and half of the warp's 32 weight rows, as tmem_ld16x16 gives them: four rows and NT / 4 tokens
  // per thread, so that a group's scales are read from shared memory a quarter as often as with a row per thread
  // (64 x 24576 x 1536: 12.7 us against 14.3)
  float acc[NT / 16][2][8];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j / 16][j / 8 % 2][j % 8] = 0.0f;

  if (warp == 4) {
    const bool leader = elect_one();
    const uint32_t at = smem_addr(smem);
    int i = 0;
    for (; i < groups; ++i) {
      const int s = i % Shape::kStages;
      if (i >= Shape::kStages && !warp_wait(&bars->empty[s], ((i / Shape::kStages) - 1) & 1, abort)) break;
      if (leader) {
        mbar_arrive_expect_tx(&bars->full[s], Shape::kStageBytes);
        tma_load_2d(at + s * Shape::kStageBytes, &map_w, (g0 + i) * kGroup, n0, &bars->full[s]);
        tma_load_2d(at + s * Shape::kStageBytes + kWTileBytes, &map_x, (g0 + i) * kGroup, t0, &bars->full[s]);
      }
      __syncwarp();
    }
    for (int j = std::max(0, i - Shape::kStages); j < i; ++j)  // every copy issued lands before the memory is reused
      mbar_wait(&bars->full[j % Shape::kStages], (j / Shape::kStages) & 1, kLinearWaitError);
  } else if (warp == 5) {
    const bool leader = elect_one();
    const uint32_t idesc = umma_idesc(128, NT, 0, false);
    const uint64_t w_desc = sw128_desc_k(smem_addr(smem)), x_desc = sw128_desc_k(smem_addr(smem) + kWTileBytes);
    for (int i = 0; i < groups; ++i) {
      const int s = i % Shape::kStages, b = i % Shape::kBufs;
      if (!warp_wait(&bars->full[s], (i / Shape::kStages) & 1, abort) ||
          (i >= Shape::kBufs && !warp_wait(&bars->sum_empty[b], ((i / Shape::kBufs) - 1) & 1, abort)))
        break;
      tc_fence_after();
      if (leader) {
        const uint64_t step = static_cast<uint64_t>(s * (Shape::kStageBytes / 16));
#pragma unroll
        for (int k = 0; k < kGroup / 32; ++k) umma_f8_ss(tmem + b * NT, w_desc + step + 2 * k, x_desc + step + 2 * k, idesc, k > 0);
        umma_commit(&bars->empty[s]);
        umma_commit(&bars->sum_full[b]);
      }
      __syncwarp();
    }
    if (leader) umma_commit(&bars->drain);
    __syncwarp();
    mbar_wait(&bars->drain, 0, kLinearWaitError);
  } else {
    // the tokens' scales, all in flight at once; a token's are consecutive
    for (int i = tid; i < NT * groups; i += 128) {
      const int t = i / groups, g = i - t * groups;
      if (t0 + t < a.rows) copy4_async(scale + g * NT + t, a.x_scales + static_cast<int64_t>(t0 + t) * groups_all + g0 + g);
      else scale[g * NT + t] = 0.0f;
    }
    const float* w_scale = a.w_scales + static_cast<int64_t>(tile) * groups_all + g0;
    float next_w = groups > 0 ? __ldg(w_scale) : 0.0f;
    copies4_wait();
    named_barrier_sync(1, 128);
    const uint32_t my_lanes = static_cast<uint32_t>(warp * kWarp) << 16;
    for (int i = 0; i < groups; ++i) {
      const int b = i % Shape::kBufs;
      const float sw = next_w;
      if (i + 1 < groups) next_w = __ldg(w_scale + i + 1);
      if (!warp_wait(&bars->sum_full[b], (i / Shape::kBufs) & 1, abort)) break;
      tc_fence_after();
      const float* f = scale + i * NT + lane % 4 * 2;
      constexpr int kAtOnce = NT < 64 ? NT : 64;
#pragma unroll
      for (int c = 0; c < NT; c += kAtOnce) {
        uint32_t d[kAtOnce / 16][2][8];
#pragma unroll
        for (int j = 0; j < kAtOnce; j += 16) {
          tmem_ld16x16(tmem + my_lanes + b * NT + c + j, d[j / 16][0]);
          tmem_ld16x16(tmem + my_lanes + (16u << 16) + b * NT + c + j, d[j / 16][1]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < kAtOnce; j += 8) {
          float2 s = *reinterpret_cast<const float2*>(f + c + j);
          s = make_float2(s.x * sw, s.y * sw);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float* sum = acc[(c + j) / 16][h] + j % 16 / 2;
            const uint32_t* v = d[j / 16][h] + j % 16 / 2;
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[q] = fmaf(__uint_as_float(v[q]), q % 2 ? s.y : s.x, sum[q]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sum_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, Shape::kCols);

  // each CTA's sums [NT][128] in its own shared memory (the pipeline's, now idle), a share of the tokens added up
  // by each CTA of the cluster
  float* part = reinterpret_cast<float*>(smem);
  if (warp < 4) {
    float* at = part + lane % 4 * 2 * kSumStride + warp * kWarp + lane / 4;
#pragma unroll
    for (int c = 0; c < NT; c += 16)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 8; ++q) at[(c + q / 4 * 8 + q % 2) * kSumStride + h * 16 + q / 2 % 2 * 8] = acc[c / 16][h][q];
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  O* out = static_cast<O*>(a.out);
  const bool whole = a.outs % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
  for (int i = tid; i < NT * 32 / splits; i += kRowsThreads) {
    const int e = i + rank * (NT * 32 / splits), t = e / 32, c = (e % 32) * 4;
    if (t0 + t >= a.rows || n0 + c >= a.outs) continue;
    float4 sum = *reinterpret_cast<const float4*>(part + t * kSumStride + c);
    if (splits > 1) {
      sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < splits; ++r) {
        const float4 v = ld_cluster(part + t * kSumStride + c, r);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
    }
    struct alignas(4 * sizeof(O)) Four {
      O v[4];
    } o{{from_float<O>(sum.x), from_float<O>(sum.y), from_float<O>(sum.z), from_float<O>(sum.w)}};
    O* to = out + static_cast<int64_t>(t0 + t) * a.outs + n0 + c;
    if (whole) {
      *reinterpret_cast<Four*>(to) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + c + j < a.outs) to[j] = o.v[j];
    }
  }
  if (splits > 1) cluster_sync();  // nobody leaves while its sums are being read
}

// ----------------------------------------------------------------- many rows

// PAIR: two CTAs (cta_group::2) take 256 tokens x TN outputs, each holding its
// 128 tokens' rows and half of the weight rows.  That halves the weights' bytes
// from L2 and runs the products faster (four steps of M = 256, N = 256 take 520
// cycles over the pair, of M = 128, N = 256 on one CTA 690).  Otherwise one CTA
// takes 128 tokens x TN.  In both a group's sums must leave tensor memory every
// 500 cycles, and the two come within a twentieth of each other per round of all
// SMs (4000 x 7168 x 16384, short runs: 458 us in pairs, 483 alone); the finer tiles of one
// CTA fill the SMs where a pair's do not (600 x 7168 x 7168: 36 us against 63).
constexpr int kTileM = 128;  // tokens per CTA
constexpr int kSumWarps = 8;  // warp w: tokens 32 (w % 4) .. + 31, half w / 4 of the TN columns
constexpr int kTilesThreads = (kSumWarps + 4) * kWarp;  // .. 8: TMA; 9, 10: the products of even and odd groups
template <int TN, bool PAIR>
struct TilesShape {
  static constexpr int kCtas = PAIR ? 2 : 1;
  static constexpr int kABytes = kTileM * kGroup, kBBytes = TN / kCtas * kGroup, kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = PAIR ? 6 : 4;
};
template <int TN, bool PAIR>
struct TilesBarriers {
  uint64_t full[TilesShape<TN, PAIR>::kStages], empty[TilesShape<TN, PAIR>::kStages];
  uint64_t sum_full[2], sum_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
template <int TN, bool PAIR>
constexpr size_t tiles_smem() {
  return 1024 + TilesShape<TN, PAIR>::kStages * TilesShape<TN, PAIR>::kStageBytes + sizeof(TilesBarriers<TN, PAIR>);
}
static_assert(tiles_smem<256, true>() <= 232448 && tiles_smem<256, false>() <= 232448, "shared memory per block");

template <typename O, int TN, bool PAIR>
__global__ void __launch_bounds__(kTilesThreads, 1)
    linear_tiles_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, LinearArgs a,
                        int m_tiles, int n_tiles) {
  using Shape = TilesShape<TN, PAIR>;
  constexpr int kStages = Shape::kStages, kHalf = TN / 2, kStageBytes = Shape::kStageBytes, kCtas = Shape::kCtas;
  extern __shared__ unsigned char smem_raw[];
  // the same place in both CTAs (their shared memory starts alike)
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto* bars = reinterpret_cast<TilesBarriers<TN, PAIR>*>(smem + kStages * kStageBytes);
  const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xFFFFFFFFu, tid / kWarp, 0);
  volatile int* abort = &bars->abort;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  const int groups = static_cast<int>((a.cols + kGroup - 1) / kGroup);
  const int tiles = m_tiles * n_tiles, pair = blockIdx.x / kCtas, pairs = gridDim.x / kCtas;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], kCtas);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->sum_full[b], 1);
      mbar_init(&bars->sum_empty[b], kCtas * kSumWarps);
    }
    mbar_init(&bars->drain, 2);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == kSumWarps + 1) {
    if (PAIR) {
      pair_tmem_alloc(&bars->tmem_base, 512);
    } else {
      tmem_alloc(&bars->tmem_base, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  // 168 registers per thread at launch (three warpgroups): the sums' two take 224
  // and the third keeps 56, 256 * 224 + 128 * 56 = 384 * 168
  if (warp >= kSumWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == kSumWarps) {
      // each CTA loads its share; the first one's barriers count both
      const bool leader = elect_one();
      const uint32_t at = smem_addr(smem), full_at = PAIR ? cluster_addr(&bars->full[0], 0) : 0;
      uint32_t i = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int m0 = (t % m_tiles * kCtas + rank) * kTileM, n0 = t / m_tiles * TN + rank * (TN / kCtas);
        for (int g = 0; g < groups; ++g, ++i) {
          const uint32_t s = i % kStages, dst = at + s * kStageBytes, bar = full_at + s * 8;
          if (i >= kStages && !warp_wait(&bars->empty[s], ((i / kStages) - 1) & 1, abort)) {
            ok = false;
            break;
          }
          if (leader) {
            if (PAIR) {
              cluster_arrive_expect_tx(bar, kStageBytes);
              pair_tma_load_2d(dst, &map_x, g * kGroup, m0, bar);
              pair_tma_load_2d(dst + Shape::kABytes, &map_w, g * kGroup, n0, bar);
            } else {
              mbar_arrive_expect_tx(&bars->full[s], kStageBytes);
              tma_load_2d(dst, &map_x, g * kGroup, m0, &bars->full[s]);
              tma_load_2d(dst + Shape::kABytes, &map_w, g * kGroup, n0, &bars->full[s]);
            }
          }
          __syncwarp();
        }
      }
      // the copies issued land before either CTA leaves: the first one's barriers count them all, and what
      // the products have consumed had landed
      for (uint32_t j = i > kStages ? i - kStages : 0; j < i; ++j)
        mbar_wait(rank == 0 ? &bars->full[j % kStages] : &bars->empty[j % kStages], (j / kStages) & 1, kLinearWaitError);
    } else if (warp == kSumWarps + 1 || warp == kSumWarps + 2) {
      // the first CTA issues, one warp per accumulator: a group's hand-over hides behind the other's
      if (rank == 0) {
        const bool leader = elect_one();
        const uint32_t b = warp - kSumWarps - 1, d = tmem + b * 256;
        const uint32_t idesc = umma_idesc(kCtas * kTileM, TN, 0, false);
        const uint64_t x_desc = sw128_desc_k(smem_addr(smem)), w_desc = sw128_desc_k(smem_addr(smem) + Shape::kABytes);
        const uint32_t mine = static_cast<uint32_t>((tiles - pair + pairs - 1) / pairs) * static_cast<uint32_t>(groups);
        auto commit = [](uint64_t* bar) {
          if (PAIR) pair_umma_commit(bar);
          else umma_commit(bar);
        };
        for (uint32_t i = b; i < mine; i += 2) {
          const uint32_t s = i % kStages;
          if (i >= 2 && !warp_wait(&bars->sum_empty[b], ((i / 2) - 1) & 1, abort)) break;
          if (!warp_wait(&bars->full[s], (i / kStages) & 1, abort)) break;
          tc_fence_after();
          if (leader) {
            const uint64_t step = static_cast<uint64_t>(s * (kStageBytes / 16));
#pragma unroll
            for (int k = 0; k < kGroup / 32; ++k) {
              if (PAIR) pair_umma_f8_ss(d, x_desc + step + 2 * k, w_desc + step + 2 * k, idesc, k > 0);
              else umma_f8_ss(d, x_desc + step + 2 * k, w_desc + step + 2 * k, idesc, k > 0);
            }
            commit(&bars->sum_full[b]);
            commit(&bars->empty[s]);
          }
          __syncwarp();
        }
        if (leader) commit(&bars->drain);
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quad = warp % 4, half = warp / 4;
    const uint32_t from = tmem + (static_cast<uint32_t>(quad * kWarp) << 16) + half * kHalf;
    const uint32_t empty_at = PAIR ? cluster_addr(&bars->sum_empty[0], 0) : 0;
    uint32_t i = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int64_t row = (t % m_tiles * kCtas + rank) * kTileM + quad * kWarp + lane;
      const int64_t n0 = static_cast<int64_t>(t / m_tiles) * TN + half * kHalf;
      // the columns from `edge` (a multiple of 16) on belong to the next 128 of the weight's rows
      const int edge = static_cast<int>(128 - n0 % 128);
      const int64_t last = (a.outs - 1) / 128;
      const float* sx = a.x_scales + std::min<int64_t>(row, a.rows - 1) * groups;
      const float* sw0 = a.w_scales + std::min<int64_t>(n0 / 128, last) * groups;
      const float* sw1 = a.w_scales + std::min<int64_t>(n0 / 128 + 1, last) * groups;
      float acc[kHalf];
#pragma unroll
      for (int j = 0; j < kHalf; ++j) acc[j] = 0.0f;
      float next0 = __ldg(sx) * __ldg(sw0), next1 = __ldg(sx) * __ldg(sw1);
      for (int g = 0; g < groups; ++g, ++i) {
        const uint32_t b = i % 2;
        const float f0 = next0, f1 = next1;
        if (g + 1 < groups) {
          const float x = __ldg(sx + g + 1);
          next0 = x * __ldg(sw0 + g + 1);
          next1 = x * __ldg(sw1 + g + 1);
        }
        if (!warp_wait(&bars->sum_full[b], (i / 2) & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // the next columns on their way while these are added; the accumulator is free once the last have left it
        uint32_t d0[32], d1[32];
        const uint32_t sums = from + b * 256;
        auto add = [&](const uint32_t (&d)[32], int c) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < kHalf) acc[(c + j) % kHalf] = fmaf(__uint_as_float(d[j]), c + j / 16 * 16 < edge ? f0 : f1, acc[(c + j) % kHalf]);
        };
        auto leave = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) cluster_arrive(empty_at + b * 8);
            else mbar_arrive(&bars->sum_empty[b]);
          }
        };
        tmem_ld32(sums, d0);
        tmem_ld_wait();
        tmem_ld32(sums + 32, d1);
        add(d0, 0);
        tmem_ld_wait();
        tmem_ld32(sums + 64, d0);
        add(d1, 32);
        tmem_ld_wait();
        if (kHalf > 112) tmem_ld32(sums + 96, d1);
        else if (kHalf > 96) tmem_ld16(sums + 96, d1);
        else leave();
        add(d0, 64);
        if (kHalf > 96) {
          tmem_ld_wait();
          leave();
          add(d1, 96);
        }
      }
      if (!ok) break;
      if (row < a.rows) {
        O* out = static_cast<O*>(a.out) + row * a.outs + n0;
        constexpr int kV = 16 / sizeof(O);
        const bool whole = n0 + kHalf <= a.outs && a.outs % kV == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
#pragma unroll
        for (int j = 0; j < kHalf; j += kV) {
          __align__(16) O v[kV];
#pragma unroll
          for (int k = 0; k < kV; ++k) v[k] = from_float<O>(acc[j + k]);
          if (whole) {
            *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<const uint4*>(v);
          } else {
#pragma unroll
            for (int k = 0; k < kV; ++k)
              if (n0 + j + k < a.outs) out[j + k] = v[k];
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // in both CTAs: every product is complete.  Only now, after the CTA's own work: the second one's products
  // warps have none, and a wait from their start on would bound the whole call, not a lack of progress.
  if (warp == kSumWarps + 1) {
    mbar_wait(&bars->drain, 0, kLinearWaitError);
    __syncwarp();
  }
  if (PAIR) cluster_sync();  // nobody leaves while the other CTA may still signal or read here
  tc_fence_after();
  if (warp == kSumWarps + 1) {
    if (PAIR) pair_tmem_dealloc(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// [rows][cols] bytes with a box of one group's columns and `box` rows, 128B-swizzled.
bool encode_codes(CUtensorMap* map, const uint8_t* base, int64_t rows, int64_t cols, int64_t stride, int box) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t boxes[2] = {kGroup, static_cast<cuuint32_t>(box)}, steps[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, boxes, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How many CTAs share a weight tile's groups: the largest cluster that keeps at least two groups per CTA and all
// CTAs resident at once (1 x 576 x 1536, 12 groups, from L2: clusters of eight 4.7 us, of four, as here, 4.7, of
// two 5.6).
template <int NT>
int rows_splits(const LinearArgs& a) {
  const int64_t tiles = ceil_div(a.outs, 128), groups = ceil_div(a.cols, kGroup), token_tiles = ceil_div(a.rows, NT);
  int splits = 1;
  while (splits < 8 && tiles * token_tiles * splits * 2 <= RowsShape<NT>::kPerSm * gemv_grid_ctas() && groups >= splits * 4) splits *= 2;
  return splits;
}
// Shared memory of a CTA, with the scales of all of its groups.
template <int NT>
size_t rows_smem_of(const LinearArgs& a) {
  return rows_smem<NT>(static_cast<int>(ceil_div(ceil_div(a.cols, kGroup), rows_splits<NT>(a))));
}

template <typename O, int NT>
cudaError_t launch_rows(const LinearArgs& a, cudaStream_t stream) {
  CUtensorMap mx, mw;
  if (!encode_codes(&mx, a.x, a.rows, a.cols, a.x_stride, NT) || !encode_codes(&mw, a.w, a.outs, a.cols, a.w_stride, 128))
    return cudaErrorInvalidValue;
  const int64_t tiles = ceil_div(a.outs, 128), groups = ceil_div(a.cols, kGroup), token_tiles = ceil_div(a.rows, NT);
  const int splits = rows_splits<NT>(a), max_groups = static_cast<int>(ceil_div(groups, splits));
  auto kernel = linear_rows_kernel<O, NT>;
  const size_t smem = rows_smem_of<NT>(a);
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(tiles * splits), static_cast<unsigned>(token_tiles));
  config.blockDim = dim3(kRowsThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(splits);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, mx, mw, a, splits, max_groups);
}

template <typename O, int TN, bool PAIR>
cudaError_t launch_tiles_n(const LinearArgs& a, cudaStream_t stream) {
  constexpr int kCtas = PAIR ? 2 : 1;
  CUtensorMap mx, mw;
  if (!encode_codes(&mx, a.x, a.rows, a.cols, a.x_stride, kTileM) || !encode_codes(&mw, a.w, a.outs, a.cols, a.w_stride, TN / kCtas))
    return cudaErrorInvalidValue;
  auto kernel = linear_tiles_kernel<O, TN, PAIR>;
  constexpr int kSmem = static_cast<int>(tiles_smem<TN, PAIR>());
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return err;
  const int64_t m_tiles = ceil_div(a.rows, kCtas * kTileM), n_tiles = ceil_div(a.outs, TN);
  if (m_tiles * n_tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(kCtas * std::min<int64_t>(m_tiles * n_tiles, gemv_grid_ctas() / kCtas)));
  config.blockDim = dim3(kTilesThreads);
  config.dynamicSmemBytes = kSmem;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCtas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, mx, mw, a, static_cast<int>(m_tiles), static_cast<int>(n_tiles));
}

// The tiles whose rounds of all SMs cover the outputs with the least work:
// 4000 x 7168 outputs are 448 tiles of a pair and 256 columns (7 rounds of 74
// pairs, the last one all but empty) or 512 of 224 (7 rounds, each an eighth
// shorter); 600 x 7168 are 140 tiles of one CTA and 256 (one round).  Narrower
// tiles of one CTA were slower than a pair's (300 x 7168 x 2048: 22 us against 16).
LinearTile many_rows_tile(const LinearArgs& a) {
  auto cost = [&](int64_t tn, int64_t ctas) {
    return ceil_div(ceil_div(a.rows, ctas * kTileM) * ceil_div(a.outs, tn), gemv_grid_ctas() / ctas) * tn;
  };
  const int64_t least = std::min({cost(256, 2), cost(224, 2), cost(192, 2), cost(256, 1)});
  if (cost(256, 2) == least) return {2 * kTileM, 256};
  if (cost(224, 2) == least) return {2 * kTileM, 224};
  if (cost(192, 2) == least) return {2 * kTileM, 192};
  return {kTileM, 256};
}

LinearTile tile_of(const LinearArgs& a) {
  // Where the scales do not fit beside the pipeline: tiles, which read them as they go.  They are slower there (100 x
  // 7168: 16384 columns 42 us, 18432, past the limit, 68).
  constexpr size_t kMost = 232448;
  if (a.rows <= 16) return rows_smem_of<16>(a) <= kMost ? LinearTile{16, 128} : many_rows_tile(a);
  if (a.rows <= 32) return rows_smem_of<32>(a) <= kMost ? LinearTile{32, 128} : many_rows_tile(a);
  if (a.rows <= 64) return rows_smem_of<64>(a) <= kMost ? LinearTile{64, 128} : many_rows_tile(a);
  // weight streaming while its CTAs can still share a group range in twos (from L2): 128 x 7168 x 2048 11.8 us against
  // 20.5 in tiles, 300 x 2112 x 7168 22.3 against 27.1; beyond that tiles: 600 x 2112 x 7168 28 against 35, 300 x 7168 x
  // 7168 32 against 66.  Over 24576 x 1536, weights from memory, where tiles begin at 65 rows: 64 rows 13.4 us, 65 rows
  // 13.5, 128 rows 16, 300 rows 25.
  if (2 * ceil_div(a.rows, 128) * ceil_div(a.outs, 128) <= gemv_grid_ctas() && rows_smem_of<128>(a) <= kMost) return {128, 128};
  return many_rows_tile(a);
}

template <typename O>
cudaError_t launch_linear(const LinearArgs& a, cudaStream_t stream) {
  const LinearTile tile = tile_of(a);
  if (tile.outs == 128) {
    switch (tile.tokens) {
      case 16: return launch_rows<O, 16>(a, stream);
      case 32: return launch_rows<O, 32>(a, stream);
      case 64: return launch_rows<O, 64>(a, stream);
      default: return launch_rows<O, 128>(a, stream);
    }
  }
  if (tile.tokens == kTileM) return launch_tiles_n<O, 256, false>(a, stream);
  switch (tile.outs) {
    case 256: return launch_tiles_n<O, 256, true>(a, stream);
    case 224: return launch_tiles_n<O, 224, true>(a, stream);
    default: return launch_tiles_n<O, 192, true>(a, stream);
  }
}

}  // namespace

cudaError_t launch_fp8_linear(const LinearArgs& a, int out_dtype, cudaStream_t stream) {
  switch (out_dtype) {
    case kDtypeF32: return launch_linear<float>(a, stream);
    case kDtypeBF16: return launch_linear<__nv_bfloat16>(a, stream);
    default: return launch_linear<__half>(a, stream);
  }
}

LinearTile fp8_linear_tile(int64_t rows, int64_t outs, int64_t cols) {
  LinearArgs a{};
  a.rows = rows; a.outs = outs; a.cols = cols;
  return tile_of(a);
}

int read_and_clear_linear_error(cudaStream_t stream) { return read_and_clear_local_error(stream); }

}  // namespace moe
