// Multi-head latent attention over a paged cache for a batch of new tokens.
//
// Append.  A token's row of the cache is its normalised latent part and its
// rotated rope part,
//   row = [ c / sqrt(mean(c^2) + eps) * w,  rot(r, position) ],
// stored at slot page * page_size + offset; the token's queries' rope parts
// are rotated by the same angles.  rot turns the pairs (2p, 2p + 1) by
// (cos[position, p], sin[position, p]).  fp32 throughout, one rounding to the
// stored type.  Bytes bound it: every value is read once and written once; a
// warp takes a token's cache row or 256 of its query values.
//
// Attention.  score[l] = scale (q_latent . c[l] + q_pe . r[l]) over the row's
// first `length` positions, position l in page table[l / page_size];
// out = sum softmax(score)[l] c[l], lse = log(sum exp(score)).  A row without
// positions gives zeros and -inf.
#include <math.h>

#include <algorithm>

#include "async_copy.cuh"
#include "fp8_gemv.cuh"
#include "plan.cuh"
#include "router.cuh"
#include "rows.cuh"
#include "serving.cuh"
#include "tcgen05.cuh"

namespace moe {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendVectors = 4;  // 8-value vectors of a latent row per lane: latent <= 1024

// The angles of the pairs at columns c, c + 2, .. of a rope group of n more columns.
struct Angles {
  float cos[4], sin[4];
};
MOE_D Angles angles_at(const float* cos, const float* sin, int c, int n) {
  Angles a;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    a.cos[p] = 2 * p < n ? __ldg(cos + c / 2 + p) : 0.0f;
    a.sin[p] = 2 * p < n ? __ldg(sin + c / 2 + p) : 0.0f;
  }
  return a;
}
template <typename T, typename C>
MOE_D Eight<C> rotated(const Eight<T>& e, const Angles& a) {
  Eight<C> r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float x = widen<T>(e.v[2 * p]), y = widen<T>(e.v[2 * p + 1]);
    r.v[2 * p] = from_float<C>(x * a.cos[p] - y * a.sin[p]);
    r.v[2 * p + 1] = from_float<C>(x * a.sin[p] + y * a.cos[p]);
  }
  return r;
}

// A CTA per token (and step): its last warp the cache row, the others the
// queries: a thread keeps its eight columns of a head, and their angles, over
// the heads that it takes, kAppendLoads of them in flight.
constexpr int kAppendLoads = 4;
template <typename T, typename W, typename C, bool VEC>
__global__ void __launch_bounds__(kAppendThreads + kWarp, 5) paged_append_kernel(AppendArgs a) {
  const int tid = threadIdx.x, q_threads = blockDim.x - kWarp, lane = tid % kWarp;
  const int latent = static_cast<int>(a.latent), rope = static_cast<int>(a.rope);
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t pos = a.positions[t];
    const bool placed = pos >= 0 && pos < a.table_rows;
    const float* cos = a.cos + (placed ? pos : 0) * (rope / 2);
    const float* sin = a.sin + (placed ? pos : 0) * (rope / 2);
    if (tid >= q_threads) {
      const int64_t slot = a.slots[t];
      if (slot < 0) continue;
      if (!placed || slot >= a.pages * a.page_size) {
        if (lane == 0) atomicOr(&g_device_error, kPagedRangeError);
        continue;
      }
      const T* src = static_cast<const T*>(a.kv) + t * a.kv_stride;
      const int64_t page = slot / a.page_size;
      C* dst = static_cast<C*>(a.cache) + page * a.page_stride + (slot - page * a.page_size) * a.row_stride;
      Eight<T> e[kAppendVectors];
      float ss = 0.0f;
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v) {
        const int c = 8 * (lane + v * kWarp), n = min(latent - c, 8);
        clear8(e[v]);
        if (n > 0) load8<T, VEC>(src + c, n, e[v]);
      }
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(widen<T>(e[v].v[j]), widen<T>(e[v].v[j]), ss);
      const float inv = 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(latent) + a.eps);
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v) {
        const int c = 8 * (lane + v * kWarp), n = min(latent - c, 8);
        if (n <= 0) break;
        Eight<W> w;
        Eight<C> o;
        load8<W, VEC>(static_cast<const W*>(a.norm_w) + c, n, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = from_float<C>(widen<T>(e[v].v[j]) * inv * widen<W>(w.v[j]));
        store8<C, VEC>(dst + c, n, o);
      }
      for (int c = 8 * lane; c < rope; c += 8 * kWarp) {
        const int n = min(rope - c, 8);
        load8<T, VEC>(src + latent + c, n, e[0]);
        store8<C, VEC>(dst + latent + c, n, rotated<T, C>(e[0], angles_at(cos, sin, c, n)));
      }
      continue;
    }
    const int per_head = (rope + 7) / 8, at_once = q_threads / per_head;  // heads at once
    if (tid >= at_once * per_head) continue;
    const int h0 = tid / per_head, c = 8 * (tid - h0 * per_head), n = min(rope - c, 8);
    const C* q = static_cast<const C*>(a.q) + t * a.q_stride + c;
    C* out = static_cast<C*>(a.q_out) + t * a.heads * rope + c;
    Eight<C> e[kAppendLoads];
    auto load = [&](int h) {
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i)
        if (h + i * at_once < a.heads) load8<C, VEC>(q + (h + i * at_once) * a.q_head_stride, n, e[i]);
    };
    load(h0);  // before the angles, which wait for the position
    const Angles turn = angles_at(cos, sin, c, n);
    for (int h = h0; h < a.heads; h += at_once * kAppendLoads) {
      if (h != h0) load(h);
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i) {
        if (h + i * at_once >= a.heads) break;
        Eight<C> o = rotated<C, C>(e[i], turn);
        if (!placed) clear8(o);  // a row that has no place in the sequence: zeros
        store8<C, VEC>(out + (h + i * at_once) * rope, n, o);
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, typename W, typename C>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
  auto whole = [](int64_t n, int64_t size) { return n * size % 16 == 0; };
  const bool vec = a.latent % 8 == 0 && a.rope % 8 == 0 && aligned16(a.kv) && whole(a.kv_stride, sizeof(T)) &&
                   aligned16(a.norm_w) && aligned16(a.cache) && whole(a.page_stride, sizeof(C)) &&
                   whole(a.row_stride, sizeof(C)) &&
                   (!a.q || (aligned16(a.q) && aligned16(a.q_out) && whole(a.q_stride, sizeof(C)) &&
                             whole(a.q_head_stride, sizeof(C))));
  const int64_t vectors = a.q ? a.heads * ceil_div(a.rope, 8) : 0;
  const int threads = static_cast<int>(std::min<int64_t>(ceil_div(vectors, kWarp) * kWarp, kAppendThreads)) + kWarp;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.tokens, INT32_MAX));
  if (vec) paged_append_kernel<T, W, C, true><<<grid, threads, 0, stream>>>(a);
  else paged_append_kernel<T, W, C, false><<<grid, threads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename C>
cudaError_t launch_append_types(const AppendArgs& a, int x_dtype, int norm_dtype, cudaStream_t stream) {
  const bool wide = norm_dtype == kDtypeF32;
  if (x_dtype == kDtypeF32)
    return wide ? launch_append<float, float, C>(a, stream) : launch_append<float, C, C>(a, stream);
  return wide ? launch_append<C, float, C>(a, stream) : launch_append<C, C, C>(a, stream);
}

// ------------------------------------------------------------- attention
//
// A CTA takes 128 heads of one row and half of the latent columns of the
// result; the two CTAs of a pair compute the same scores.  Tensor memory holds
// the 128 x 256 fp32 result, two 128 x 64 score tiles (the softmax of one while
// the other is computed; its 16-bit probabilities replace the scores) and 256
// columns of the queries: all 512 columns.  Shared memory holds the queries'
// other columns (80 KiB) and the cache rows in chunks of 64 positions x 64
// columns (8 KiB, 128B-swizzled): the chunks of this CTA's own columns stay
// until the second product has read them (3 tiles of them), the others pass
// through 6 slots as the scores are computed.
//   scores  S = Q K^T:  M = 128 heads, N = 64 positions, k over the columns
//   result  O += P V:   M = 128 heads, N = own columns, k over the positions;
// V is the same shared memory as K, read as an MN-major operand.
// Halving the columns costs the scores twice (832 instead of 544 multiply-adds
// per head and position and CTA) but leaves room in tensor memory for the
// overlap; the cache is read from memory once, the pair's second read hits L2.
//
// The softmax's reference maximum moves only when a tile's maximum exceeds it
// by 2^8 (log2 domain): probabilities stay below 2^8 of the reference's 1, well
// inside 16-bit range, and the 256 columns of the result are rescaled rarely.
// Probabilities are rounded to the cache's type for the second product, half a
// step each; their sum is of the unrounded fp32 values.
//
// Work: all rows' tiles of 64 positions in one sequence, cut into equal
// ranges, one per CTA pair, so that lengths need not be alike.  A row inside
// one range is finished there; a row that is cut leaves fp32 parts in the
// workspace, which the second kernel joins.  A range has at most two parts.
//
// Warps 0-3: softmax, result (a thread per head).  4-7: the cache's rows.
// 8: tensor memory and the products (the whole warp walks the work, so that
// operand descriptors stay in uniform registers; one lane issues).
//
// Rows arrive by TMA, one box per chunk and run of positions that no page
// border cuts (gcd(page size, 64) of them), or, where such runs are shorter than
// 8, by 16-byte asynchronous copies of four warps.  Positions that do not take
// part (past the length, or on a page outside the cache) are masked in the scores;
// their rows may hold anything, NaN among it, so the softmax warps clear them
// in shared memory before the second product reads them with probability 0.
constexpr int kTile = 64;
constexpr int kHeads = 128;
constexpr int kChunkBytes = kTile * 128;
constexpr int kQChunkBytes = kHeads * 128;
constexpr int kQTmemChunks = 4, kQSmemChunks = 5;
constexpr int kKeptStages = 3, kKeptChunks = 4;
constexpr int kPassing = 6;
constexpr int kSoftmaxThreads = 128, kCopyThreads = 128;
constexpr int kAttnThreads = kSoftmaxThreads + kCopyThreads + kWarp;
constexpr int kAttnWarps = kAttnThreads / kWarp;
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 384;
constexpr int kMinTiles = 2;  // fewest tiles worth a range of their own
constexpr float kMovesBy = 8.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnBarriers {
  uint64_t kept_full[kKeptStages], kept_empty[kKeptStages];
  uint64_t pass_full[kPassing], pass_empty[kPassing];
  uint64_t s_full[2];    // scores complete
  uint64_t p_ready[2];   // probabilities written (one arrival per softmax warp)
  uint64_t q_ready;      // queries of the next part in place
  uint64_t o_done;       // a tile's second product complete
  uint64_t o_read;       // the part's result has been read
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int first_item, first_tile;
  long long sums[kAttnWarps];
};
constexpr size_t kAttnSmem = 1024 + static_cast<size_t>(kQSmemChunks) * kQChunkBytes +
                             static_cast<size_t>(kKeptStages * kKeptChunks + kPassing) * kChunkBytes + sizeof(AttnBarriers);
static_assert(kAttnSmem <= 232448, "shared memory per block");

struct AttnPlan {
  float* part_o;       // [2 workers][128 heads][latent]: unnormalised
  float2* part_ml;     // [2 workers][128 heads]: reference maximum (log2 domain), sum
  int64_t* before;     // [batch + 1]: tiles before each row
  int workers;         // pairs of CTAs
  int run;             // positions per TMA box
  int groups;          // groups of 128 heads: an item is a row's group
};

MOE_HD int64_t range_start(int64_t w, int64_t total, int64_t workers) { return w * total / workers; }
MOE_D int64_t used_workers(int64_t total, int64_t workers) {
  return max(int64_t(1), min(workers, total / kMinTiles));
}

MOE_D int row_length(const PagedAttnArgs& a, int64_t b) {
  const int64_t room = a.table_cols * a.page_size;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > room ? static_cast<int>(room) : n;
}
MOE_D int tiles_of(int len) { return (len + kTile - 1) / kTile; }

// The parts of a range in order; every role walks them by itself.
struct Part {
  int64_t b;
  int group, tile0, tiles, len;
  bool whole;
  int slot;
};
struct Walk {
  int64_t item;
  int tile0;
  int64_t left;
  MOE_D bool next(const PagedAttnArgs& a, int groups, int worker, Part& p) {
    if (left <= 0) return false;
    int n;
    while (true) {
      p.b = item / groups;
      p.len = row_length(a, p.b);
      n = tiles_of(p.len) - tile0;
      if (n > 0) break;
      ++item;
      tile0 = 0;
    }
    p.group = static_cast<int>(item - p.b * groups);
    p.tile0 = tile0;
    p.tiles = static_cast<int>(min(static_cast<int64_t>(n), left));
    p.whole = tile0 == 0 && p.tiles == n;
    p.slot = 2 * worker + (tile0 > 0 ? 0 : 1);
    left -= p.tiles;
    ++item;
    tile0 = 0;
    return true;
  }
};

MOE_D float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T>
MOE_D uint32_t pack2(float lo, float hi);
template <>
MOE_D uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
MOE_D uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

MOE_D void copy16(uint32_t dst, const void* src, bool present) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(present ? 16 : 0) : "memory");
}
MOE_D void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// A wait of a whole warp: every lane sees the same answer.
MOE_D bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int code) {
  return __all_sync(0xFFFFFFFFu, wait_or_abort(bar, parity, abort, code));
}

template <typename T, bool TMA>
__global__ void __launch_bounds__(kAttnThreads, 1) paged_attention_kernel(const __grid_constant__ CUtensorMap map_cache,
                                                                          const __grid_constant__ CUtensorMap map_ql,
                                                                          const __grid_constant__ CUtensorMap map_qp,
                                                                          PagedAttnArgs a, AttnPlan plan) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_smem = smem;
  unsigned char* kept_smem = q_smem + kQSmemChunks * kQChunkBytes;
  unsigned char* pass_smem = kept_smem + kKeptStages * kKeptChunks * kChunkBytes;
  AttnBarriers* bars = reinterpret_cast<AttnBarriers*>(pass_smem + kPassing * kChunkBytes);
  const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xFFFFFFFFu, tid / kWarp, 0);
  volatile int* abort = &bars->abort;
  const int latent = static_cast<int>(a.latent), rope = static_cast<int>(a.rope);
  const int lat_chunks = (latent + 63) / 64, chunks = lat_chunks + 1;  // the last one holds the rope part
  const int halves = lat_chunks > 1 ? 2 : 1, per_half = (lat_chunks + halves - 1) / halves;
  const int worker = blockIdx.x / halves, half = blockIdx.x % halves;
  const int kept0 = half * per_half, kept_n = min(per_half, lat_chunks - kept0);
  const int q_tmem = min(kQTmemChunks, lat_chunks);

  // tiles before each thread's rows; the range's first item
  long long mine = 0;
  const int64_t per = ceil_div(a.batch, kAttnThreads), b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
  for (int64_t b = b0; b < b1; ++b) mine += static_cast<long long>(tiles_of(row_length(a, b))) * plan.groups;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < kWarp; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == kWarp - 1) bars->sums[warp] = upto;
  __syncthreads();
  long long before = upto - mine, total = 0;
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += bars->sums[w];
    total += bars->sums[w];
  }
  if (blockIdx.x == 0) {
    long long at = before;
    for (int64_t b = b0; b < b1; ++b) {
      plan.before[b] = at;
      at += static_cast<long long>(tiles_of(row_length(a, b))) * plan.groups;
      if (a.lengths[b] > a.table_cols * a.page_size) atomicOr(&g_device_error, kPagedRangeError);
    }
    if (tid == 0) plan.before[a.batch] = total;
  }
  const int64_t workers = used_workers(total, plan.workers);
  if (worker >= workers || total == 0) return;
  const int64_t start = range_start(worker, total, workers), stop = range_start(worker + 1, total, workers);
  if (start >= before && start < before + mine) {
    long long at = before;
    int64_t item = b0 * plan.groups;
    while (true) {
      const int n = tiles_of(row_length(a, item / plan.groups));
      if (start < at + n) break;
      at += n;
      ++item;
    }
    bars->first_item = static_cast<int>(item);
    bars->first_tile = static_cast<int>(start - at);
  }
  if (tid == 0) {
    for (int s = 0; s < kKeptStages; ++s) {
      mbar_init(&bars->kept_full[s], TMA ? 1 : kCopyThreads);
      mbar_init(&bars->kept_empty[s], 1);
    }
    for (int s = 0; s < kPassing; ++s) {
      mbar_init(&bars->pass_full[s], TMA ? 1 : kCopyThreads);
      mbar_init(&bars->pass_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->p_ready[s], kSoftmaxThreads / kWarp);
    }
    mbar_init(&bars->q_ready, kSoftmaxThreads / kWarp + 1);
    mbar_init(&bars->o_done, 1);
    mbar_init(&bars->o_read, kSoftmaxThreads / kWarp);
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == kAttnWarps - 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  Walk walk{bars->first_item, bars->first_tile, stop - start};
  Part p;

  if (TMA && warp >= kSoftmaxThreads / kWarp && warp < kAttnWarps - 1) {
    // --------------------------------------------------------------- TMA
    if (warp == kSoftmaxThreads / kWarp) {
      const uint32_t kept_at = smem_addr(kept_smem), pass_at = smem_addr(pass_smem);
      const int run = plan.run, runs = kTile / run, page_size = static_cast<int>(a.page_size);
      const bool leader = elect_one();
      uint32_t g = 0, pc = 0, kept = 0;
      bool ok = true;
      // lane r: the page of the tile's run r (-1: none) and its first row there
      auto lookup = [&](int tile, int& page, int& row) {
        const int pos = tile * kTile + lane * run;
        page = -1;
        row = 0;
        if (lane < runs && pos < p.len) {
          const int col = pos / page_size;
          page = __ldg(a.table + p.b * a.table_stride + col);
          row = pos - col * page_size;
          if (page >= a.pages) page = -1;
        }
      };
      while (ok && walk.next(a, plan.groups, worker, p)) {
        int page, row, next_page = -1, next_row = 0;
        lookup(p.tile0, page, row);
        for (int i = 0; i < p.tiles && ok; ++i, ++g) {
          if (i + 1 < p.tiles) lookup(p.tile0 + i + 1, next_page, next_row);
          const int present = __popc(__ballot_sync(0xFFFFFFFFu, page >= 0));
          auto fetch = [&](int c, uint32_t dst, uint64_t* bar) {
            const int x = c < lat_chunks ? c * 64 : latent;
            for (int r = 0; r < runs; ++r) {
              const int pg = __shfl_sync(0xFFFFFFFFu, page, r), at = __shfl_sync(0xFFFFFFFFu, row, r);
              if (pg >= 0 && leader) tma_load_3d(dst + r * run * 128, &map_cache, x, at, pg, bar);
            }
          };
          const int s = g % kKeptStages;
          if (g >= kKeptStages && !warp_wait(&bars->kept_empty[s], ((g / kKeptStages) - 1) & 1, abort, kPagedWaitError)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&bars->kept_full[s], present * run * 128 * kept_n);
          __syncwarp();
          ++kept;
          for (int k = 0; k < kept_n; ++k) fetch(kept0 + k, kept_at + (s * kKeptChunks + k) * kChunkBytes, &bars->kept_full[s]);
          for (int c = 0; c < chunks; ++c) {
            if (c >= kept0 && c < kept0 + kept_n) continue;
            const int slot = pc % kPassing;
            if (pc >= kPassing && !warp_wait(&bars->pass_empty[slot], ((pc / kPassing) - 1) & 1, abort, kPagedWaitError)) {
              ok = false;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&bars->pass_full[slot], present * run * 128);
            __syncwarp();
            fetch(c, pass_at + slot * kChunkBytes, &bars->pass_full[slot]);
            ++pc;
          }
          page = next_page;
          row = next_row;
        }
      }
      // every copy issued lands before the CTA may exit
      for (uint32_t j = kept > kKeptStages ? kept - kKeptStages : 0; j < kept; ++j)
        mbar_wait(&bars->kept_full[j % kKeptStages], (j / kKeptStages) & 1, kPagedWaitError);
      for (uint32_t j = pc > kPassing ? pc - kPassing : 0; j < pc; ++j)
        mbar_wait(&bars->pass_full[j % kPassing], (j / kPassing) & 1, kPagedWaitError);
    }
  } else if (!TMA && warp >= kSoftmaxThreads / kWarp && warp < kAttnWarps - 1) {
    // ------------------------------------------------------------ copies
    const int ct = tid - kSoftmaxThreads, unit = ct % 8, row0 = ct / 8;
    const uint32_t kept_at = smem_addr(kept_smem), pass_at = smem_addr(pass_smem);
    uint32_t g = 0, pc = 0;
    bool ok = true;
    while (ok && walk.next(a, plan.groups, worker, p)) {
      const int32_t* table = a.table + p.b * a.table_stride;
      for (int i = 0; i < p.tiles && ok; ++i, ++g) {
        const T* src[4];
        bool live[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int pos = (p.tile0 + i) * kTile + row0 + 16 * j;
          src[j] = static_cast<const T*>(a.cache);
          live[j] = pos < p.len;
          if (live[j]) {
            const int col = pos / static_cast<int>(a.page_size);
            const int page = __ldg(table + col);
            live[j] = page >= 0 && page < a.pages;
            if (live[j]) src[j] += page * a.page_stride + (pos - col * static_cast<int>(a.page_size)) * a.row_stride;
          }
        }
        // chunk c: columns 64 c .. of the latent part, or the rope part
        auto fetch = [&](int c, uint32_t dst) {
          const int col = (c < lat_chunks ? c * 64 : latent) + unit * 8;
          const bool in = c < lat_chunks ? col < latent : unit * 8 < rope;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = row0 + 16 * j;
            copy16(dst + r * 128 + ((unit ^ (r % 8)) * 16), src[j] + (in ? col : 0), live[j] && in);
          }
        };
        const int s = g % kKeptStages;
        if (g >= kKeptStages && !wait_or_abort(&bars->kept_empty[s], ((g / kKeptStages) - 1) & 1, abort, kPagedWaitError)) {
          ok = false;
          break;
        }
        for (int k = 0; k < kept_n; ++k) fetch(kept0 + k, kept_at + (s * kKeptChunks + k) * kChunkBytes);
        copies_arrive(&bars->kept_full[s]);
        for (int c = 0; c < chunks; ++c) {
          if (c >= kept0 && c < kept0 + kept_n) continue;
          const int slot = pc % kPassing;
          if (pc >= kPassing && !wait_or_abort(&bars->pass_empty[slot], ((pc / kPassing) - 1) & 1, abort, kPagedWaitError)) {
            ok = false;
            break;
          }
          fetch(c, pass_at + slot * kChunkBytes);
          copies_arrive(&bars->pass_full[slot]);
          ++pc;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kAttnWarps - 1) {
    // ---------------------------------------------------------- products
    const bool leader = elect_one();
    const int format = __is_same(T, __nv_bfloat16) ? 1 : 0;
    const uint32_t idesc_s = umma_idesc(kHeads, kTile, format, false);
    const uint32_t idesc_o = umma_idesc(kHeads, 64 * kept_n, format, true);
    const uint64_t q_desc = sw128_desc_k(smem_addr(q_smem)), k_desc = sw128_desc_k(smem_addr(kept_smem));
    const uint64_t pass_desc = sw128_desc_k(smem_addr(pass_smem)), v_desc = sw128_desc(smem_addr(kept_smem), kChunkBytes);
    uint32_t g = 0, pc = 0, parts = 0;
    bool ok = true;
    // descriptors advance in units of 16 bytes: 2 per 16 columns of a swizzled row
    auto chunk_scores = [&](int c, uint64_t b, uint32_t d, bool first) {
      if (c < q_tmem) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16_ts(d, tmem + kColQ + c * 32 + k * 8, b + 2 * k, idesc_s, !(first && k == 0));
      } else {
        const uint64_t q = q_desc + (c - q_tmem) * (kQChunkBytes / 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16_ss(d, q + 2 * k, b + 2 * k, idesc_s, !(first && k == 0));
      }
    };
    // the scores of the tile whose number is t
    auto scores = [&](uint32_t t) {
      const uint32_t s = t % kKeptStages, d = tmem + kColS + (t % 2) * kTile;
      if (!warp_wait(&bars->kept_full[s], (t / kKeptStages) & 1, abort, kPagedWaitError)) return false;
      if (!TMA) fence_proxy_async_shared();
      tc_fence_after();
      for (int k = 0; k < kept_n; ++k)
        if (leader) chunk_scores(kept0 + k, k_desc + (s * kKeptChunks + k) * (kChunkBytes / 16), d, k == 0);
      for (int c = 0; c < chunks; ++c) {
        if (c >= kept0 && c < kept0 + kept_n) continue;
        const uint32_t slot = pc % kPassing;
        if (!warp_wait(&bars->pass_full[slot], (pc / kPassing) & 1, abort, kPagedWaitError)) return false;
        if (!TMA) fence_proxy_async_shared();
        tc_fence_after();
        if (leader) {
          chunk_scores(c, pass_desc + slot * (kChunkBytes / 16), d, false);
          umma_commit(&bars->pass_empty[slot]);
        }
        __syncwarp();
        ++pc;
      }
      if (leader) umma_commit(&bars->s_full[t % 2]);
      __syncwarp();
      return true;
    };
    while (ok && walk.next(a, plan.groups, worker, p)) {
      const int tiles = __shfl_sync(0xFFFFFFFFu, p.tiles, 0);
      if (!warp_wait(&bars->q_ready, parts & 1, abort, kPagedWaitError)) break;
      tc_fence_after();
      ok = scores(g);
      for (int i = 0; i < tiles && ok; ++i, ++g) {
        if (i + 1 < tiles && !(ok = scores(g + 1))) break;
        if (!(ok = warp_wait(&bars->p_ready[g % 2], (g / 2) & 1, abort, kPagedWaitError))) break;
        if (i == 0 && parts > 0 && !(ok = warp_wait(&bars->o_read, (parts - 1) & 1, abort, kPagedWaitError))) break;
        tc_fence_after();
        const uint32_t s = g % kKeptStages;
        if (leader) {
          const uint64_t v = v_desc + s * (kKeptChunks * kChunkBytes / 16);
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            umma_f16_ts(tmem + kColO, tmem + kColS + (g % 2) * kTile + k * 8, v + k * (2048 / 16), idesc_o, i > 0 || k > 0);
          umma_commit(&bars->kept_empty[s]);
          umma_commit(&bars->o_done);
        }
        __syncwarp();
      }
      ++parts;
    }
    if (leader) umma_commit(&bars->drain);  // every product issued is complete before tensor memory is freed
    __syncwarp();
    mbar_wait(&bars->drain, 0, kPagedWaitError);
  } else {
    // ------------------------------------------------- softmax and result
    const float c2 = fmaxf(a.scale * kLog2e, 1e-37f);  // above 0: a masked score's -inf stays one
    const uint32_t my_lanes = static_cast<uint32_t>(warp * kWarp) << 16;
    const int page_size = static_cast<int>(a.page_size);
    // the part's queries: columns from 64 q_tmem on by TMA (absent heads and columns arrive as zeros), the others a
    // thread its own row, all loads in flight together
    auto load_queries = [&](const Part& p) {
      const int h0 = p.group * kHeads, nh = static_cast<int>(min(a.heads - h0, static_cast<int64_t>(kHeads)));
      if (tid == 0) {
        mbar_arrive_expect_tx(&bars->q_ready, (chunks - q_tmem) * kQChunkBytes);
        for (int c = q_tmem; c < chunks; ++c)
          tma_load_3d(smem_addr(q_smem) + (c - q_tmem) * kQChunkBytes, c < lat_chunks ? &map_ql : &map_qp,
                      c < lat_chunks ? c * 64 : 0, h0, static_cast<int>(p.b), &bars->q_ready);
      }
      __syncwarp();
      const T* ql = static_cast<const T*>(a.q_latent) + p.b * a.ql_stride + (h0 + tid) * a.ql_head_stride;
      __align__(16) uint32_t v[kQTmemChunks][32];
#pragma unroll
      for (int c = 0; c < kQTmemChunks; ++c)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int col = c * 64 + u * 8;
          *reinterpret_cast<uint4*>(v[c] + 4 * u) = tid < nh && c < q_tmem && col < latent
                                                        ? __ldg(reinterpret_cast<const uint4*>(ql + col))
                                                        : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int c = 0; c < kQTmemChunks; ++c) tmem_st32(tmem + my_lanes + kColQ + c * 32, v[c]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_ready);
    };
    uint32_t g = 0;
    bool ok = true, more = walk.next(a, plan.groups, worker, p);
    if (more) load_queries(p);
    while (ok && more) {
      float m = -INFINITY, l = 0.0f;
      const int32_t* table = a.table + p.b * a.table_stride;
      for (int i = 0; i < p.tiles; ++i, ++g) {
        // positions that take part: inside the length, on a page of the cache
        uint32_t live[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int pos = (p.tile0 + i) * kTile + k * kWarp + lane;
          bool in = pos < p.len;
          if (in) {
            const int page = __ldg(table + pos / page_size);
            in = page >= 0 && page < a.pages;
            if (!in) atomicOr(&g_device_error, kPagedRangeError);
          }
          live[k] = __ballot_sync(0xFFFFFFFFu, in);
        }
        if (!warp_wait(&bars->s_full[g % 2], (g / 2) & 1, abort, kPagedWaitError)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t s_at = tmem + my_lanes + kColS + (g % 2) * kTile;
        uint32_t r[kTile];
        tmem_ld32(s_at, r);
        tmem_ld32(s_at + 32, r + 32);
        tmem_ld_wait();
        if ((live[0] & live[1]) != 0xFFFFFFFFu) {
#pragma unroll
          for (int j = 0; j < kTile; ++j)
            if (!(live[j / 32] >> (j % 32) & 1u)) r[j] = 0xFF800000u;  // -inf
          if (TMA) {  // the scores are complete: nothing reads these rows now but the second product
            unsigned char* v_at = kept_smem + (g % kKeptStages) * kKeptChunks * kChunkBytes;
            for (int row = tid / 8; row < kTile; row += kSoftmaxThreads / 8)
              if (!(live[row / 32] >> (row % 32) & 1u))
                for (int k = 0; k < kept_n; ++k)
                  *reinterpret_cast<uint4*>(v_at + k * kChunkBytes + row * 128 + (tid % 8) * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_shared();
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kTile; ++j) top = fmaxf(top, __uint_as_float(r[j]));
        top *= c2;
        const bool moves = top > m + kMovesBy || (m == -INFINITY && top > m);
        if (__any_sync(0xFFFFFFFFu, moves)) {
          const float f = !moves ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - top);
          if (moves) {
            l *= f;
            m = top;
          }
          if (i > 0) {
            if (!warp_wait(&bars->o_done, (g - 1) & 1, abort, kPagedWaitError)) {
              ok = false;
              break;
            }
            tc_fence_after();
            for (int c = 0; c < 64 * kept_n; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem + my_lanes + kColO + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st32(tmem + my_lanes + kColO + c, o);
            }
            tmem_st_wait();
          }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int j = 0; j < kTile; j += 2) {
          const float p0 = exp2_fast(fmaf(__uint_as_float(r[j]), c2, -ref));
          const float p1 = exp2_fast(fmaf(__uint_as_float(r[j + 1]), c2, -ref));
          sum0 += p0;
          sum1 += p1;
          r[j / 2] = pack2<T>(p0, p1);
        }
        l += sum0 + sum1;
        tmem_st32(s_at, r);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_ready[g % 2]);
      }
      if (!ok) break;
      const Part done = p;
      more = walk.next(a, plan.groups, worker, p);
      if (more) load_queries(p);  // the last scores are complete: the queries' places are free
      if (!warp_wait(&bars->o_done, (g - 1) & 1, abort, kPagedWaitError)) break;
      tc_fence_after();
      const int64_t h = done.group * kHeads + tid;
      const bool has = h < a.heads;
      const int col0 = kept0 * 64, cols = min(64 * kept_n, latent - col0);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      T* out = static_cast<T*>(a.out) + (done.b * a.heads + h) * latent + col0;
      float* part = plan.part_o + (static_cast<int64_t>(done.slot) * kHeads + tid) * latent + col0;
      for (int c = 0; c < cols; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem + my_lanes + kColO + c, o);
        tmem_ld_wait();
        if (!has) continue;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (c + j >= cols) break;
          if (done.whole) {
            uint4 v;
            v.x = pack2<T>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv);
            v.y = pack2<T>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            v.z = pack2<T>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
            v.w = pack2<T>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
            *reinterpret_cast<uint4*>(out + c + j) = v;
          } else {
            *reinterpret_cast<uint4*>(part + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            *reinterpret_cast<uint4*>(part + c + j + 4) = make_uint4(o[j + 4], o[j + 5], o[j + 6], o[j + 7]);
          }
        }
      }
      if (half == 0 && has) {
        if (!done.whole) plan.part_ml[static_cast<int64_t>(done.slot) * kHeads + tid] = make_float2(m, l);
        else if (a.lse) a.lse[done.b * a.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->o_read);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kAttnWarps - 1) tmem_dealloc(tmem, 512);
}

// Joins the parts of the rows that were cut, and writes the rows without
// positions.  A CTA takes two heads of a row; a thread four columns.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(PagedAttnArgs a, AttnPlan plan) {
  const int64_t pairs = ceil_div(a.heads, 2);
  const int64_t b = blockIdx.x / pairs, h = (blockIdx.x - b * pairs) * 2 + threadIdx.x / (kJoinThreads / 2);
  if (h >= a.heads) return;
  const int64_t c = 4 * (threadIdx.x % (kJoinThreads / 2));
  const bool in = c < a.latent;
  const int64_t total = plan.before[a.batch], tiles = (plan.before[b + 1] - plan.before[b]) / plan.groups;
  T* out = static_cast<T*>(a.out) + (b * a.heads + h) * a.latent + c;
  if (tiles == 0) {
    if (in) *reinterpret_cast<uint2*>(out) = make_uint2(0, 0);
    if (a.lse && c == 0) a.lse[b * a.heads + h] = -INFINITY;
    return;
  }
  const int64_t workers = used_workers(total, plan.workers), group = h / kHeads;
  const int64_t t0 = plan.before[b] + group * tiles, t1 = t0 + tiles - 1;  // the item's first and last tile
  const int64_t w0 = ((t0 + 1) * workers - 1) / total, w1 = ((t1 + 1) * workers - 1) / total;
  if (w0 == w1) return;  // finished where it was computed
  // the first part is its range's last (unless the range starts with the row), the others open theirs
  auto at = [&](int64_t w) { return (2 * w + (w == w0 ? 1 : 0)) * kHeads + (h - group * kHeads); };
  float top = -INFINITY;
  for (int64_t w = w0; w <= w1; ++w) top = fmaxf(top, plan.part_ml[at(w)].x);
  if (top == -INFINITY) top = 0.0f;
  float sum = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int64_t w = w0; w <= w1; ++w) {
    const float2 ml = plan.part_ml[at(w)];
    const float f = exp2_fast(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    if (in) {
      const float4 o = *reinterpret_cast<const float4*>(plan.part_o + at(w) * a.latent + c);
      acc.x = fmaf(o.x, f, acc.x);
      acc.y = fmaf(o.y, f, acc.y);
      acc.z = fmaf(o.z, f, acc.z);
      acc.w = fmaf(o.w, f, acc.w);
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (in) *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  if (a.lse && c == 0) a.lse[b * a.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

AttnPlan attn_plan(Plan& p, int64_t batch, int64_t heads, int64_t latent, int64_t table_cols, int64_t page_size) {
  AttnPlan l{};
  const int64_t halves = latent > 64 ? 2 : 1;
  l.groups = static_cast<int>(ceil_div(heads, kHeads));
  // at most one pair of CTAs per pair of SMs, and no more than there can be ranges
  const int64_t most = batch * l.groups * ceil_div(table_cols * page_size, kTile);
  l.workers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(gemv_grid_ctas() / halves, ceil_div(most, kMinTiles))));
  l.run = 1;
  while (l.run < kTile && page_size % (2 * l.run) == 0) l.run *= 2;
  l.part_o = p.take<float>(2 * l.workers * kHeads * latent);
  l.part_ml = p.take<float2>(2 * l.workers * kHeads);
  l.before = p.take<int64_t>(batch + 1);
  return l;
}

// A tensor [z][y][x] of 16-bit values with a box of 64 columns and `rows` rows, 128B-swizzled.
template <typename T>
bool encode_rows(CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int64_t y_stride, int64_t z_stride,
                 int rows) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  // a dimension of one has no stride of its own, but the map wants one
  if (y == 1) y_stride = 64;
  if (z == 1) z_stride = 64;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(x), static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(y_stride) * 2, static_cast<cuuint64_t>(z_stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(rows), 1}, steps[3] = {1, 1, 1};
  return encode(map, __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
cudaError_t launch_attention(const PagedAttnArgs& a, const AttnPlan& plan, cudaStream_t stream) {
  const bool tma = plan.run >= 8;
  CUtensorMap cache{}, ql, qp;
  if (!encode_rows<T>(&ql, a.q_latent, a.latent, a.heads, a.batch, a.ql_head_stride, a.ql_stride, kHeads) ||
      !encode_rows<T>(&qp, a.q_pe, a.rope, a.heads, a.batch, a.qp_head_stride, a.qp_stride, kHeads) ||
      (tma && !encode_rows<T>(&cache, a.cache, a.latent + a.rope, a.page_size, a.pages, a.row_stride, a.page_stride, plan.run)))
    return cudaErrorInvalidValue;
  auto kernel = tma ? paged_attention_kernel<T, true> : paged_attention_kernel<T, false>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kAttnSmem));
  if (err != cudaSuccess) return err;
  const unsigned ctas = static_cast<unsigned>(plan.workers * (a.latent > 64 ? 2 : 1));
  kernel<<<ctas, kAttnThreads, kAttnSmem, stream>>>(cache, ql, qp, a, plan);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  paged_attention_join_kernel<T><<<static_cast<unsigned>(a.batch * ceil_div(a.heads, 2)), kJoinThreads, 0, stream>>>(a, plan);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs& a, int x_dtype, int norm_dtype, int cache_dtype, cudaStream_t stream) {
  if (cache_dtype == kDtypeBF16) return launch_append_types<__nv_bfloat16>(a, x_dtype, norm_dtype, stream);
  return launch_append_types<__half>(a, x_dtype, norm_dtype, stream);
}

int64_t paged_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t latent, int64_t table_cols, int64_t page_size) {
  Plan p;
  attn_plan(p, batch, heads, latent, table_cols, page_size);
  return static_cast<int64_t>(p.used());
}

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, char* workspace, cudaStream_t stream) {
  Plan p(workspace);
  const AttnPlan plan = attn_plan(p, a.batch, a.heads, a.latent, a.table_cols, a.page_size);
  return dtype == kDtypeBF16 ? launch_attention<__nv_bfloat16>(a, plan, stream) : launch_attention<__half>(a, plan, stream);
}

int read_and_clear_paged_error(cudaStream_t stream) { return read_and_clear_local_error(stream); }

}  // namespace moe
