// Multi-head latent attention over a paged cache for a batch of new tokens.
//
// Append.  A token's row of the cache is its normalised latent part and its
// rotated rope part,
//   row = [ c / sqrt(mean(c^2) + eps) * w,  rot(r, position) ],
// stored at slot page * page_size + offset; the token's queries' rope parts
// are rotated by the same angles.  rot turns the pairs (2p, 2p + 1) by
// (cos[position, p], sin[position, p]).  fp32 throughout, one rounding to the
// stored type.  Bytes bound it: every value is read once and written once; a
// warp takes a token's cache row or 256 of its query values.  Measured with 128
// heads, inputs from memory: 4096 tokens 26.6 us (145 MB, 5.4 TB/s), 32 tokens 3.6 us
// (2.8 from L2).
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
template <bool VEC>
MOE_D Angles angles_at(const float* cos, const float* sin, int c, int n) {
  Angles a;
  if (VEC) {  // whole and aligned, like the values
    const float4 k = __ldg(reinterpret_cast<const float4*>(cos + c / 2)), s = __ldg(reinterpret_cast<const float4*>(sin + c / 2));
    a.cos[0] = k.x, a.cos[1] = k.y, a.cos[2] = k.z, a.cos[3] = k.w;
    a.sin[0] = s.x, a.sin[1] = s.y, a.sin[2] = s.z, a.sin[3] = s.w;
    return a;
  }
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

// A CTA takes tokens in turn: its last warp the cache rows, the others the
// queries: a thread keeps its eight columns of a head, and their angles, over the
// heads that it takes, kAppendLoads of them in flight, and asks for the next
// token's first ones before it turns this token's.  Three CTAs per SM: 4096
// tokens of 128 heads 26.4 us; four, where registers run short, 34, two 31, and a
// CTA per token without the loads ahead 35.
constexpr int kAppendLoads = 4, kAppendCtas = 3;
template <typename T, typename W, typename C, bool VEC>
__global__ void __launch_bounds__(kAppendThreads + kWarp, kAppendCtas) paged_append_kernel(AppendArgs a) {
  const int tid = threadIdx.x, q_threads = blockDim.x - kWarp, lane = tid % kWarp;
  const int latent = static_cast<int>(a.latent), rope = static_cast<int>(a.rope);
  auto in_table = [&](int64_t pos) { return pos >= 0 && pos < a.table_rows; };
  if (tid >= q_threads) {
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
      const T* src = static_cast<const T*>(a.kv) + t * a.kv_stride;
      const int64_t pos = a.positions[t], slot = a.slots[t];
      Eight<T> e[kAppendVectors], r;
      const int r_col = 8 * lane, r_n = min(rope - r_col, 8);
      clear8(r);
      if (r_n > 0) load8<T, VEC>(src + latent + r_col, r_n, r);
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v) {
        const int c = 8 * (lane + v * kWarp), n = min(latent - c, 8);
        clear8(e[v]);
        if (n > 0) load8<T, VEC>(src + c, n, e[v]);
      }
      if (slot < 0) continue;
      if (!in_table(pos) || slot >= a.pages * a.page_size) {
        if (lane == 0) atomicOr(&g_device_error, kPagedRangeError);
        continue;
      }
      const float* cos = a.cos + pos * (rope / 2);
      const float* sin = a.sin + pos * (rope / 2);
      const int64_t page = slot / a.page_size;
      C* dst = static_cast<C*>(a.cache) + page * a.page_stride + (slot - page * a.page_size) * a.row_stride;
      float ss = 0.0f;
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
      for (int c = r_col, n = r_n; n > 0;) {
        store8<C, VEC>(dst + latent + c, n, rotated<T, C>(r, angles_at<VEC>(cos, sin, c, n)));
        c += 8 * kWarp;
        n = min(rope - c, 8);
        if (n > 0) load8<T, VEC>(src + latent + c, n, r);
      }
    }
    return;
  }
  const int per_head = (rope + 7) / 8, at_once = q_threads / per_head;  // heads at once
  if (tid >= at_once * per_head) return;
  const int h0 = tid / per_head, c = 8 * (tid - h0 * per_head), n = min(rope - c, 8);
  auto load = [&](int64_t t, int h, Eight<C> (&e)[kAppendLoads]) {
    const C* q = static_cast<const C*>(a.q) + t * a.q_stride + c;
#pragma unroll
    for (int i = 0; i < kAppendLoads; ++i)
      if (h + i * at_once < a.heads) load8<C, VEC>(q + (h + i * at_once) * a.q_head_stride, n, e[i]);
  };
  Eight<C> e[kAppendLoads], ahead[kAppendLoads];
  int64_t t = blockIdx.x, pos = a.positions[t], pos_ahead = 0;
  load(t, h0, e);  // before the angles, which wait for the position
  for (; t < a.tokens; t += gridDim.x) {
    const bool placed = in_table(pos);
    const int64_t row = (placed ? pos : 0) * (rope / 2);
    const Angles turn = angles_at<VEC>(a.cos + row, a.sin + row, c, n);
    if (t + gridDim.x < a.tokens) {
      pos_ahead = a.positions[t + gridDim.x];
      load(t + gridDim.x, h0, ahead);
    }
    C* out = static_cast<C*>(a.q_out) + t * a.heads * rope + c;
    for (int h = h0; h < a.heads; h += at_once * kAppendLoads) {
      if (h != h0) load(t, h, e);
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i) {
        if (h + i * at_once >= a.heads) break;
        Eight<C> o = rotated<C, C>(e[i], turn);
        if (!placed) clear8(o);  // a row that has no place in the sequence: zeros
        store8<C, VEC>(out + (h + i * at_once) * rope, n, o);
      }
    }
    pos = pos_ahead;
#pragma unroll
    for (int i = 0; i < kAppendLoads; ++i) e[i] = ahead[i];
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, typename W, typename C>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
  auto whole = [](int64_t n, int64_t size) { return n * size % 16 == 0; };
  const bool vec = a.latent % 8 == 0 && a.rope % 8 == 0 && aligned16(a.cos) && aligned16(a.sin) && aligned16(a.kv) && whole(a.kv_stride, sizeof(T)) &&
                   aligned16(a.norm_w) && aligned16(a.cache) && whole(a.page_stride, sizeof(C)) &&
                   whole(a.row_stride, sizeof(C)) &&
                   (!a.q || (aligned16(a.q) && aligned16(a.q_out) && whole(a.q_stride, sizeof(C)) &&
                             whole(a.q_head_stride, sizeof(C))));
  const int64_t vectors = a.q ? a.heads * ceil_div(a.rope, 8) : 0;
  const int threads = static_cast<int>(std::min<int64_t>(ceil_div(vectors, kWarp) * kWarp, kAppendThreads)) + kWarp;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.tokens, kAppendCtas * gemv_grid_ctas()));
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
// A pair of CTAs takes 128 heads of one row, 64 each, as one tcgen05.mma
// cta_group::2 product with M = 128 over the pair:
//   scores  S = Q K^T:  N = 128 positions (64 from each CTA), k over the columns
//   result  O += P V:   N = 256 latent columns (128 from each CTA), k over the
//                       positions, twice for 512 columns
// At M = 128 a pair's product costs N / 4 cycles (measured: 34 at N = 128, 66 at
// N = 256), all of the tensor cores' rate; one CTA alone with M = 128 needs
// 76 cycles at N = 64 and has no room in tensor memory for 512 columns of result.
// In tensor memory a CTA's 64 heads lie in lanes 0-63 with the first half of N
// and in lanes 64-127 with the second: a softmax thread holds 64 positions of
// one head, and shares the head's maximum and sum with the thread 64 further.
//
// Shared memory: the queries (9 chunks of 64 heads x 64 columns, 8 KiB), the
// probabilities (16-bit, 16 KiB), and a buffer for each of a tile's five loads,
// in chunks of 64 positions x 64 columns (128B-swizzled): K's columns 0-255,
// 256-511 and rope (64 positions, half of the tile), V's own 256 columns of the
// tile's first and second half (the same rows again, from L2, as an MN-major
// operand).  Each is loaded again as soon as the products have read it, a whole
// tile ahead of its next use.  Bytes bound it: a position's 1152 bytes come from
// memory once per 128 heads.
//
// The softmax's reference maximum moves only when a tile's maximum exceeds it
// by 2^8 (log2 domain): probabilities stay below 2^8 of the reference's 1, well
// inside 16-bit range, and the result is rescaled rarely.  Probabilities are
// rounded to the cache's type for the second product, half a step each; their
// sum is of the unrounded fp32 values.
//
// Work: all rows' tiles of 128 positions in one sequence, cut into equal
// ranges, one per pair of CTAs, so that lengths need not be alike.  A row
// inside one range is finished there; a row that is cut leaves fp32 parts in
// the workspace, which the second kernel joins.  A range has at most two parts.
//
// Rows arrive by TMA, one box per run of positions that no page border cuts (the
// largest power of two, up to 64, that divides the page size).  A copy costs the
// issuing warp some 90 cycles, so full buffers take four chunks with each: runs
// of 64 in the order [chunk][64 rows], shorter ones in blocks of 8 positions,
// [8 rows of a chunk][4 chunks], an order that the operands' descriptors can
// follow too (128 rows of 16 heads on 16-position pages: 90 us with 8-row blocks,
// 113 with a copy per chunk and 16 rows).  The scores of positions that do not
// take part are masked; their rows of V must not hold a NaN all the same.  Runs
// without a position, or on a page outside the cache, arrive as zeros, from
// coordinates outside the tensor; the rows of a run behind the length that cuts
// it (whatever their memory holds) are cleared in shared memory before the
// products may read.
//
// Warps 0-3: softmax, result.  4: copies of queries and K.  5, 6: copies of V's
// halves.  7: tensor memory and, in the first CTA, the products (the whole warp
// walks the work, so that operand descriptors stay in uniform registers; one
// lane issues).
//
// Measured, bf16, cache from memory: 64 rows of 128 heads and up to 8192 positions
// 114 us in a loop of a second (393 MB, 3.5 TB/s; 91 GFLOP, 0.80 PFLOP/s, at the
// 1700 MHz that the power limit leaves), 106 us after a rest.  A tile of a pair takes
// some 3350 cycles, 2280 of them products, with 16 heads as with 128 and from
// L2 as from memory; the parts' results and their join take some 12 us.  One row of
// 4096 positions 18.8 us, 16.5 from L2: launches, two tiles per pair, and the join
// of its parts.
constexpr int kTile = 128, kHalfTile = 64;
constexpr int kHeads = 128, kCtaHeads = 64;
constexpr int kChunkBytes = 64 * 128;
constexpr int kQChunks = 9;
constexpr int kBuffers = 5;  // K columns 0-255, 256-511, rope; V of the first and the second half of the tile
constexpr int kBufferChunk[kBuffers] = {0, 4, 8, 9, 13};  // where each starts, in chunks
constexpr int kBufferChunks = 17;
constexpr int kPBytes = 2 * kChunkBytes;
constexpr int kSoftmaxWarps = 4, kSoftmaxThreads = kSoftmaxWarps * kWarp;
constexpr int kKeysWarp = 4, kValuesWarp = 5, kProductsWarp = 7;
constexpr int kAttnWarps = 8, kAttnThreads = kAttnWarps * kWarp;
constexpr uint32_t kColO = 0, kColS = 256;
constexpr int kMinTiles = 2;  // fewest tiles worth a range of their own: one row of 4096 positions, from L2, 16.7 us, 1 would take 17.9
constexpr float kMovesBy = 8.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnBarriers {
  uint64_t full[kBuffers];   // of the first CTA: both CTAs' copies of a buffer have been issued, and their bytes
  uint64_t empty[kBuffers];  // in both
  uint64_t q_full;          // of the first CTA: both CTAs' queries of a part
  uint64_t s_full[2];       // scores complete
  uint64_t p_ready;         // of the first CTA: probabilities written (one arrival per softmax warp of both)
  uint64_t pv_done;         // a tile's second product complete
  uint64_t o_read;          // of the first CTA: the part's result has been read
  uint64_t cut[2];          // the bytes of a half of V that the length cuts
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int first_item, first_tile;
  long long sums[kAttnWarps];
  float share[2][kSoftmaxThreads];  // what the two threads of a head tell each other
};
constexpr size_t kAttnSmem = 1024 + static_cast<size_t>(kQChunks + kBufferChunks) * kChunkBytes + kPBytes +
                             sizeof(AttnBarriers);
static_assert(kAttnSmem <= 232448, "shared memory per block");

struct AttnPlan {
  float* part_o;       // [2 workers][latent / 8][128 heads][8]: unnormalised; a warp stores 32 heads' sectors side by side
  float2* part_ml;     // [2 workers][128 heads]: reference maximum (log2 domain), sum
  int64_t* before;     // [batch + 1]: tiles before each row
  int workers;         // pairs of CTAs
  int run;             // positions per TMA box
  int shift, page_size;  // log2 of the page size where it has one, else -1
  bool wide;           // full buffers by boxes of four chunks, each of `run` (64 or 8) positions
  int groups;          // groups of 128 heads: an item is a row's group
};

MOE_D int page_of(const AttnPlan& plan, int pos) { return plan.shift >= 0 ? pos >> plan.shift : pos / plan.page_size; }

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

// 32 bytes, 32-byte aligned.
MOE_D void store_sector(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
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

// A wait of a whole warp: every lane sees the same answer.
MOE_D bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xFFFFFFFFu, wait_or_abort(bar, parity, abort, kPagedWaitError));
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kAttnThreads, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap map_wide, const __grid_constant__ CUtensorMap map_runs,
                           const __grid_constant__ CUtensorMap map_ql, const __grid_constant__ CUtensorMap map_qp,
                           PagedAttnArgs a, AttnPlan plan) {
  extern __shared__ unsigned char smem_raw[];
  // the same place in both CTAs (their shared memory starts alike)
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_smem = smem;
  unsigned char* p_smem = q_smem + kQChunks * kChunkBytes;
  unsigned char* buffers = p_smem + kPBytes;
  AttnBarriers* bars = reinterpret_cast<AttnBarriers*>(buffers + kBufferChunks * kChunkBytes);
  const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xFFFFFFFFu, tid / kWarp, 0);
  volatile int* abort = &bars->abort;
  const int latent = static_cast<int>(a.latent), rope = static_cast<int>(a.rope);
  const int lat_chunks = (latent + 63) / 64, chunks = lat_chunks + 1;  // the last one holds the rope part
  const int own_chunks = (lat_chunks + 1) / 2;                         // latent chunks whose V each CTA brings
  const int v_pairs = (own_chunks + 1) / 2;                            // .. two at a time: a product of N = 256
  const uint32_t rank = cluster_rank();
  const int worker = blockIdx.x / 2;

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
  if (worker >= workers || total == 0) return;  // both CTAs of the pair alike
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
    for (int s = 0; s < kBuffers; ++s) {
      mbar_init(&bars->full[s], 2);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->cut[0], 1);
    mbar_init(&bars->cut[1], 1);
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->s_full[0], 1);
    mbar_init(&bars->s_full[1], 1);
    mbar_init(&bars->p_ready, 2 * kSoftmaxWarps);
    mbar_init(&bars->pv_done, 1);
    mbar_init(&bars->o_read, 2 * kSoftmaxWarps);
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == kProductsWarp) pair_tmem_alloc(&bars->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  Walk walk{bars->first_item, bars->first_tile, stop - start};
  Part p;

  if (warp >= kKeysWarp && warp < kProductsWarp) {
    // ------------------------------------------------------------ copies
    const uint32_t buffers_at = smem_addr(buffers), q_at = smem_addr(q_smem), full_at = cluster_addr(&bars->full[0], 0);
    const int run = plan.run, runs = kHalfTile / run;
    const int outside = static_cast<int>(a.pages);  // a page that the cache does not have: zeros
    const bool leader = elect_one(), wide = plan.wide, blocks = wide && run < kHalfTile;
    uint32_t g = 0, parts = 0;
    bool ok = true;
    // Where 64 positions lie: run `lane` (and lane + 32, where there are 64 runs of one position), its page as the
    // table has it (-1: none; looked at when it is used, a tile later); the run that the length cuts is whole here, and
    // positions from `dead` on do not take part.
    struct Half {
      int page, row, page2, row2, dead;
    };
    auto lookup = [&](int pos0) {
      Half r;
      auto find = [&](int i, int& page, int& row) {
        const int pos = pos0 + i * run, col = page_of(plan, pos);
        page = -1;
        row = pos - col * static_cast<int>(a.page_size);
        if (i < runs && pos < p.len) page = __ldg(a.table + p.b * a.table_stride + col);
      };
      r.page2 = -1;
      r.row2 = 0;
      if (runs > kWarp) find(lane + kWarp, r.page2, r.row2);
      find(lane, r.page, r.row);
      r.dead = max(0, p.len - pos0);
      return r;
    };
    // absent runs: a page that the cache does not have, zeros
    auto known = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(outside) ? page : outside; };
    // 64 positions of `n` chunks from the c-th on into dst
    auto copy = [&](uint32_t dst, const Half& r, int c, int n, uint32_t bar) {
      if (wide && n == 4) {
        if (lane < runs) pair_tma_load_4d(dst + lane * 4096, &map_wide, 0, r.row, c, known(r.page), bar);
        return;
      }
      const int page = known(r.page), page2 = known(r.page2);
      for (int k = 0; k < n; ++k) {
        const int x = c == lat_chunks ? latent : (c + k) * 64;
        const uint32_t to = dst + k * kChunkBytes;
        if (lane < runs) pair_tma_load_3d(to + lane * run * 128, &map_runs, x, r.row, page, bar);
        if (runs > kWarp) pair_tma_load_3d(to + (lane + kWarp) * 128, &map_runs, x, r.row2, page2, bar);
      }
    };
    uint32_t cuts = 0;
    // buffer i (chunks from first_chunk on) gets chunks c .. c + n - 1 of 64 positions, in tile g, once its memory is
    // free; each CTA tells the first one's barrier, which expects both CTAs' bytes
    auto fill = [&](int i, int first_chunk, const Half& r, int c, int n) {
      if (g >= 1 && !warp_wait(&bars->empty[i], (g - 1) & 1, abort)) return false;
      const uint32_t dst = buffers_at + first_chunk * kChunkBytes, bar = full_at + i * 8;
      const uint32_t bytes = static_cast<uint32_t>(n) * kChunkBytes;
      const bool clear = i >= 3 && r.dead > 0 && r.dead % run != 0 && r.dead < kHalfTile;
      if (!clear) {
        // (each CTA adds its own bytes: a remote arrival may come before or after the bytes that it announces)
        if (leader) cluster_arrive_expect_tx(bar, bytes);
        __syncwarp();
        copy(dst, r, c, n, bar);
        __syncwarp();
        return true;
      }
      uint64_t* own = &bars->cut[i - 3];
      if (leader) mbar_arrive_expect_tx(own, bytes);
      __syncwarp();
      copy(dst, r, c, n, cluster_addr(own, rank));
      __syncwarp();
      if (!warp_wait(own, cuts & 1, abort)) return false;
      ++cuts;
      unsigned char* at = buffers + first_chunk * kChunkBytes;
      const bool in_blocks = blocks && n == 4;
      const int chunk_bytes = in_blocks ? 1024 : kChunkBytes, atom_bytes = in_blocks ? 4096 : 1024;
      for (int row = r.dead + lane / 8; row < (r.dead + run - 1) / run * run; row += 4)
        for (int k = 0; k < n; ++k)
          *reinterpret_cast<uint4*>(at + k * chunk_bytes + row / 8 * atom_bytes + row % 8 * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_shared();
      __syncwarp();
      if (leader) cluster_arrive(bar);
      __syncwarp();
      return true;
    };
    if (warp == kKeysWarp) {
      const int half = static_cast<int>(rank) * kHalfTile, k0 = min(4, lat_chunks);
      while (ok && walk.next(a, plan.groups, worker, p)) {
        if (parts > 0 && !(ok = warp_wait(&bars->s_full[(g - 1) % 2], ((g - 1) / 2) & 1, abort))) break;  // the queries' last use
        if (leader) {
          const uint32_t bar = cluster_addr(&bars->q_full, 0);
          if (rank == 0) mbar_arrive_expect_tx(&bars->q_full, 2 * chunks * kChunkBytes);
          for (int c = 0; c < chunks; ++c)
            pair_tma_load_3d(q_at + c * kChunkBytes, c < lat_chunks ? &map_ql : &map_qp, c < lat_chunks ? c * 64 : 0,
                             p.group * kHeads + static_cast<int>(rank) * kCtaHeads, static_cast<int>(p.b), bar);
        }
        __syncwarp();
        Half now = lookup(p.tile0 * kTile + half);
        for (int i = 0; i < p.tiles && ok; ++i, ++g) {
          ok = fill(0, 0, now, 0, k0) && (lat_chunks <= 4 || fill(1, 4, now, 4, lat_chunks - 4)) && fill(2, 8, now, lat_chunks, 1);
          if (i + 1 < p.tiles) now = lookup((p.tile0 + i + 1) * kTile + half);
        }
        ++parts;
      }
    } else {
      const int c = static_cast<int>(rank) * own_chunks, h = warp - kValuesWarp;
      while (ok && walk.next(a, plan.groups, worker, p)) {
        Half now = lookup(p.tile0 * kTile + h * kHalfTile);
        for (int i = 0; i < p.tiles && ok; ++i, ++g) {
          ok = fill(3 + h, 9 + 4 * h, now, c, own_chunks);
          if (i + 1 < p.tiles) now = lookup((p.tile0 + i + 1) * kTile + h * kHalfTile);
        }
      }
    }
    // the copies issued land before either CTA leaves: the first one's barriers count them all, and what
    // the products have consumed had landed
    if (g > 0)
      for (int i = warp == kKeysWarp ? 0 : warp - kValuesWarp + 3, n = warp == kKeysWarp ? 3 : i + 1; i < n; ++i)
        if (i != 1 || lat_chunks > 4)
          mbar_wait(rank == 0 ? &bars->full[i] : &bars->empty[i], (g - 1) & 1, kPagedWaitError);
  } else if (warp == kProductsWarp) {
    // ---------------------------------------------------------- products
    if (rank == 0) {
      const bool leader = elect_one();
      const int format = __is_same(T, __nv_bfloat16) ? 1 : 0;
      const uint32_t idesc_s = umma_idesc(kHeads, kTile, format, false), idesc_o = umma_idesc(kHeads, 256, format, true);
      const uint64_t q_desc = sw128_desc_k(smem_addr(q_smem)), p_desc = sw128_desc_k(smem_addr(p_smem));
      // buffers in blocks of 8 positions, where they hold four chunks
      const bool blocks = plan.wide && plan.run < kHalfTile, v_blocks = blocks && own_chunks == 4;
      const uint64_t k_desc = sw128_desc_k(smem_addr(buffers)), block_desc = sw128_desc_k(smem_addr(buffers), 4096);
      const uint32_t v_at = smem_addr(buffers) + kBufferChunk[3] * kChunkBytes;
      const uint64_t v_desc = v_blocks ? sw128_desc(v_at, 1024, 4096) : sw128_desc(v_at, kChunkBytes);
      constexpr int kStep = kChunkBytes / 16;  // descriptors advance in units of 16 bytes
      const int v_chunk = v_blocks ? 64 : kStep, v_step = v_blocks ? 2 * 4096 / 16 : 2 * 1024 / 16;  // the next chunk, 16 positions
      uint32_t g = 0, parts = 0;
      bool ok = true;
      // the scores of the tile whose number is t
      auto scores = [&](uint32_t t) {
        const uint32_t d = tmem + kColS + (t % 2) * (kTile / 2);
        for (int i = 0; i < 3; ++i) {
          if (i == 1 && lat_chunks <= 4) continue;
          const int c0 = i == 2 ? lat_chunks : 4 * i, n = i == 2 ? 1 : min(4, lat_chunks - c0);
          if (!warp_wait(&bars->full[i], t & 1, abort)) return false;
          tc_fence_after();
          if (leader) {
            const bool in_blocks = blocks && n == 4;
            const uint64_t k0 = (in_blocks ? block_desc : k_desc) + 4 * i * kStep;
            const int k_chunk = in_blocks ? 64 : kStep;
            for (int c = 0; c < n; ++c) {
              const uint64_t q = q_desc + (c0 + c) * kStep, k = k0 + c * k_chunk;
#pragma unroll
              for (int j = 0; j < 4; ++j) pair_umma_f16_ss(d, q + 2 * j, k + 2 * j, idesc_s, i > 0 || c > 0 || j > 0);
            }
            pair_umma_commit(&bars->empty[i]);
            if (i == 2) pair_umma_commit(&bars->s_full[t % 2]);
          }
          __syncwarp();
        }
        return true;
      };
      while (ok && walk.next(a, plan.groups, worker, p)) {
        const int tiles = __shfl_sync(0xFFFFFFFFu, p.tiles, 0);
        if (!warp_wait(&bars->q_full, parts & 1, abort)) break;
        ok = scores(g);
        for (int i = 0; i < tiles && ok; ++i, ++g) {
          if (i + 1 < tiles && !(ok = scores(g + 1))) break;
          if (!(ok = warp_wait(&bars->p_ready, g & 1, abort))) break;
          if (i == 0 && parts > 0 && !(ok = warp_wait(&bars->o_read, (parts - 1) & 1, abort))) break;
          for (int h = 0; h < 2; ++h) {
            if (!(ok = warp_wait(&bars->full[3 + h], g & 1, abort))) break;
            tc_fence_after();
            if (leader) {
              for (int j = 0; j < v_pairs; ++j) {
                const uint64_t pd = p_desc + h * kStep, v = v_desc + 4 * h * kStep + 2 * j * v_chunk;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  pair_umma_f16_ss(tmem + kColO + j * 128, pd + 2 * k, v + k * v_step, idesc_o, i > 0 || h > 0 || k > 0);
              }
              pair_umma_commit(&bars->empty[3 + h]);
              if (h == 1) pair_umma_commit(&bars->pv_done);
            }
            __syncwarp();
          }
        }
        ++parts;
      }
      if (leader) pair_umma_commit(&bars->drain);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------- softmax and result
    const float c2 = fmaxf(a.scale * kLog2e, 1e-37f);  // above 0: a masked score's -inf stays one
    const uint32_t my_lanes = static_cast<uint32_t>(warp * kWarp) << 16;
    const int head = tid % kCtaHeads, part_of = tid / kCtaHeads;  // the thread's head of the CTA, and half of N
    const uint32_t ready_at = cluster_addr(&bars->p_ready, 0);
    const uint32_t read_at = cluster_addr(&bars->o_read, 0);
    int turn = 0;
    // the value of this thread's head in the other half; `fine` becomes whether it is for all four warps, so
    // that after a wait that ran out they leave together
    auto other = [&](float v, bool& fine) {
      bars->share[turn][tid] = v;
      uint32_t all;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.and.pred p, 1, %2, q;\n selp.u32 %0, 1, 0, p;\n}"
          : "=r"(all)
          : "r"(static_cast<uint32_t>(fine)), "n"(kSoftmaxThreads)
          : "memory");
      fine = all != 0;
      const float got = bars->share[turn][tid ^ kCtaHeads];
      turn ^= 1;
      return got;
    };
    uint32_t g = 0;
    bool ok = true;
    while (ok && walk.next(a, plan.groups, worker, p)) {
      float m = -INFINITY, l = 0.0f;
      const int32_t* table = a.table + p.b * a.table_stride;
      for (int i = 0; i < p.tiles; ++i, ++g) {
        // positions that take part: inside the length, on a page of the cache
        uint32_t live[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int pos = (p.tile0 + i) * kTile + part_of * kHalfTile + k * kWarp + lane;
          bool in = pos < p.len;
          if (in) {
            const int page = __ldg(table + page_of(plan, pos));
            in = page >= 0 && page < a.pages;
            if (!in) atomicOr(&g_device_error, kPagedRangeError);
          }
          live[k] = __ballot_sync(0xFFFFFFFFu, in);
        }
        bool got = ok && warp_wait(&bars->s_full[g % 2], (g / 2) & 1, abort);
        tc_fence_after();
        uint32_t r[kHalfTile];
        tmem_ld32(tmem + my_lanes + kColS + (g % 2) * kHalfTile, r);
        tmem_ld32(tmem + my_lanes + kColS + (g % 2) * kHalfTile + 32, r + 32);
        tmem_ld_wait();
        if ((live[0] & live[1]) != 0xFFFFFFFFu) {
#pragma unroll
          for (int j = 0; j < kHalfTile; ++j)
            if (!(live[j / 32] >> (j % 32) & 1u)) r[j] = 0xFF800000u;  // -inf
        }
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < kHalfTile; j += 2) {
          t0 = fmaxf(t0, __uint_as_float(r[j]));
          t1 = fmaxf(t1, __uint_as_float(r[j + 1]));
        }
        float top = fmaxf(t0, t1);
        top = fmaxf(top, other(top, got)) * c2;
        if (!got) {
          ok = false;
          break;
        }
        const bool moves = top > m + kMovesBy || (m == -INFINITY && top > m);
        if (__any_sync(0xFFFFFFFFu, moves)) {
          const float f = !moves ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - top);
          if (moves) {
            l *= f;
            m = top;
          }
          if (i > 0) {
            ok = warp_wait(&bars->pv_done, (g - 1) & 1, abort);  // (a failure shows in the next wait of all)
            tc_fence_after();
            for (int c = 0; c < v_pairs * 128; c += 32) {
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
        for (int j = 0; j < kHalfTile; j += 2) {
          const float p0 = exp2_fast(fmaf(__uint_as_float(r[j]), c2, -ref));
          const float p1 = exp2_fast(fmaf(__uint_as_float(r[j + 1]), c2, -ref));
          sum0 += p0;
          sum1 += p1;
          r[j / 2] = pack2<T>(p0, p1);
        }
        l += sum0 + sum1;
        if (g > 0) ok = warp_wait(&bars->pv_done, (g - 1) & 1, abort) && ok;  // the last probabilities have been read
        unsigned char* dst = p_smem + part_of * kChunkBytes + head * 128;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          *reinterpret_cast<uint4*>(dst + ((u ^ (head % 8)) * 16)) = make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]);
        fence_proxy_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cluster_arrive(ready_at);
      }
      ok = ok && warp_wait(&bars->pv_done, (g - 1) & 1, abort);
      const float sum = l + other(l, ok);
      if (!ok) break;
      tc_fence_after();
      // a thread its head's columns of this half of N, whole 32-byte sectors at a time
      const float scale = p.whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
      const int row = static_cast<int>(rank) * kCtaHeads + head;  // of the group's 128 heads
      const bool has = row < a.heads - p.group * kHeads;
      T* out = static_cast<T*>(a.out) + (p.b * a.heads + p.group * kHeads + row) * latent;
      const bool sectors = latent % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0;
      float* part = plan.part_o + static_cast<int64_t>(p.slot) * kHeads * latent + row * 8;
      for (int c = 0; c < own_chunks; ++c) {  // 64 columns
        const int col0 = (part_of * own_chunks + c) * 64;
        if (col0 >= latent) break;
        uint32_t o[64];
        tmem_ld32(tmem + my_lanes + kColO + c * 64, o);
        tmem_ld32(tmem + my_lanes + kColO + c * 64 + 32, o + 32);
        tmem_ld_wait();
        if (!has) continue;
#pragma unroll
        for (int j = 0; j < 64; j += 16) {
          if (col0 + j >= latent) break;
          if (!p.whole) {
            store_sector(part + (col0 + j) * kHeads, o + j);
            if (col0 + j + 8 < latent) store_sector(part + (col0 + j + 8) * kHeads, o + j + 8);
            continue;
          }
          uint32_t v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[k] = pack2<T>(__uint_as_float(o[j + 2 * k]) * scale, __uint_as_float(o[j + 2 * k + 1]) * scale);
          if (sectors && col0 + j + 16 <= latent) store_sector(out + col0 + j, v);
          else {
            *reinterpret_cast<uint4*>(out + col0 + j) = make_uint4(v[0], v[1], v[2], v[3]);
            if (col0 + j + 8 < latent) *reinterpret_cast<uint4*>(out + col0 + j + 8) = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      const int64_t h = p.group * kHeads + static_cast<int64_t>(rank) * kCtaHeads + head;
      if (part_of == 0 && h < a.heads) {
        if (!p.whole) plan.part_ml[static_cast<int64_t>(p.slot) * kHeads + (h - p.group * kHeads)] = make_float2(m, sum);
        else if (a.lse) a.lse[p.b * a.heads + h] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * kLn2;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) cluster_arrive(read_at);
    }
  }
  tc_fence_before();
  __syncthreads();
  // in both CTAs: every product is complete.  Only now, after the CTA's own work: the second one's products
  // warp has none, and a wait from its start on would bound the whole call, not a lack of progress.
  if (warp == kProductsWarp) {
    mbar_wait(&bars->drain, 0, kPagedWaitError);
    __syncwarp();
  }
  cluster_sync();  // nobody leaves while the other CTA may still signal or read here
  tc_fence_after();
  if (warp == kProductsWarp) pair_tmem_dealloc(tmem, 512);
}

MOE_D void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Joins the parts of the rows that were cut, and writes the rows without
// positions.  A CTA takes kJoinHeads heads of a row (of one group), a thread one
// of them and half of every (64 / kJoinHeads)-th block of eight columns; the
// parts' weights first, all at once, then their columns with eight loads in
// flight: four blocks of two parts and four heads where there are many rows,
// each cut into two or three parts (64 rows of 128 heads and 4096 positions
// 67.5 us against 75.7 with one head per CTA, 24 rows 36.7 against 40.0), and eight
// parts of one head where there are few (one row 16.7 us against 21.2, 4 rows
// 23.0 against 26.8; 16 rows 33.5 against 32.5).
constexpr int kJoinThreads = 128, kMostWorkers = 128;
template <typename T, int kJoinHeads>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(PagedAttnArgs a, AttnPlan plan) {
  __shared__ float weight[kJoinHeads][kMostWorkers], total_of[kJoinHeads], ref_of[kJoinHeads];
  const int per_row = static_cast<int>(ceil_div(a.heads, kJoinHeads));
  const int64_t b = blockIdx.x / per_row, h0 = static_cast<int64_t>(blockIdx.x - b * per_row) * kJoinHeads;
  const int heads = static_cast<int>(min(a.heads - h0, static_cast<int64_t>(kJoinHeads)));
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  constexpr int kBlocks = kJoinThreads / 2 / kJoinHeads;  // of eight columns, at once
  const int head = threadIdx.x / 2 % kJoinHeads, c0 = threadIdx.x / (2 * kJoinHeads) * 8 + threadIdx.x % 2 * 4;
  auto in = [&](int i) { return head < heads && c0 + i * kBlocks * 8 < a.latent; };
  wait_for_previous_kernel();
  const int64_t total = plan.before[a.batch], first = plan.before[b], next = plan.before[b + 1];
  T* out = static_cast<T*>(a.out) + (b * a.heads + h0 + head) * a.latent + c0;
  if (first == next) {
    for (int i = 0; i < kJoinHeads; ++i)
      if (in(i)) *reinterpret_cast<uint2*>(out + i * kBlocks * 8) = make_uint2(0, 0);
    if (a.lse && threadIdx.x < heads) a.lse[b * a.heads + h0 + threadIdx.x] = -INFINITY;
    return;
  }
  const int64_t workers = used_workers(total, plan.workers), group = h0 / kHeads, tiles = (next - first) / plan.groups;
  const int64_t t0 = first + group * tiles, t1 = t0 + tiles - 1;  // the item's first and last tile
  const int w0 = static_cast<int>(((t0 + 1) * workers - 1) / total), w1 = static_cast<int>(((t1 + 1) * workers - 1) / total);
  if (w0 == w1) return;  // finished where it was computed
  // the first part is its range's last, the others open theirs
  const int64_t row0 = h0 - group * kHeads;
  auto slot = [&](int w) { return (2 * static_cast<int64_t>(w) + (w == w0 ? 1 : 0)) * kHeads; };
  for (int h = warp; h < heads; h += kJoinThreads / kWarp) {
    float2 ml[kMostWorkers / kWarp];
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kMostWorkers / kWarp; ++k) {
      const int w = w0 + k * kWarp + lane;
      ml[k] = w <= w1 ? plan.part_ml[slot(w) + row0 + h] : make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, ml[k].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < kMostWorkers / kWarp; ++k) {
      const float e = exp2_fast(ml[k].x - ref);
      weight[h][k * kWarp + lane] = e;
      sum += e * ml[k].y;
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      total_of[h] = sum;
      ref_of[h] = ref;
    }
  }
  __syncthreads();
  float4 acc[kJoinHeads];  // of the thread's blocks
#pragma unroll
  for (int i = 0; i < kJoinHeads; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kAtOnce = 8 / kJoinHeads;  // parts
  const int64_t from = static_cast<int64_t>(c0 / 8) * kHeads * 8 + (row0 + head) * 8 + c0 % 8;
  for (int w = w0; w <= w1; w += kAtOnce) {
    float4 o[kAtOnce][kJoinHeads];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
      for (int i = 0; i < kJoinHeads; ++i)
        o[k][i] = w + k <= w1 && in(i) ? __ldcg(reinterpret_cast<const float4*>(plan.part_o + slot(w + k) * a.latent + from + i * kBlocks * 8 * kHeads))
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (w + k > w1) break;
      const float e = weight[head][w + k - w0];
#pragma unroll
      for (int i = 0; i < kJoinHeads; ++i) {
        acc[i].x = fmaf(o[k][i].x, e, acc[i].x);
        acc[i].y = fmaf(o[k][i].y, e, acc[i].y);
        acc[i].z = fmaf(o[k][i].z, e, acc[i].z);
        acc[i].w = fmaf(o[k][i].w, e, acc[i].w);
      }
    }
  }
  const float inv = total_of[head] == 0.0f ? 0.0f : 1.0f / total_of[head];
#pragma unroll
  for (int i = 0; i < kJoinHeads; ++i)
    if (in(i)) *reinterpret_cast<uint2*>(out + i * kBlocks * 8) = make_uint2(pack2<T>(acc[i].x * inv, acc[i].y * inv), pack2<T>(acc[i].z * inv, acc[i].w * inv));
  if (a.lse && threadIdx.x < heads)
    a.lse[b * a.heads + h0 + threadIdx.x] =
        total_of[threadIdx.x] == 0.0f ? -INFINITY : (ref_of[threadIdx.x] + log2f(total_of[threadIdx.x])) * kLn2;
}

AttnPlan attn_plan(Plan& p, int64_t batch, int64_t heads, int64_t latent, int64_t table_cols, int64_t page_size) {
  AttnPlan l{};
  l.groups = static_cast<int>(ceil_div(heads, kHeads));
  // at most one pair of CTAs per pair of SMs, and no more than there can be ranges
  const int64_t most = batch * l.groups * ceil_div(table_cols * page_size, kTile);
  l.workers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({gemv_grid_ctas() / 2, kMostWorkers, ceil_div(most, kMinTiles)})));
  l.run = 1;
  while (l.run < kHalfTile && page_size % (2 * l.run) == 0) l.run *= 2;
  l.page_size = static_cast<int>(page_size);
  l.shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == int64_t(1) << i) l.shift = i;
  // four chunks at a time need whole chunks, and pay where there are four: up to 256 latent columns V has two
  l.wide = l.run >= 8 && latent % 64 == 0 && latent > 256;
  if (l.wide && l.run < kHalfTile) l.run = 8;
  l.part_o = p.take<float>(2 * l.workers * kHeads * latent);
  l.part_ml = p.take<float2>(2 * l.workers * kHeads);
  l.before = p.take<int64_t>(batch + 1);
  return l;
}

// A tensor [z][y][x] of 16-bit values with a box of 64 columns and `rows` rows, 128B-swizzled; or, with
// `chunks`, its first 64 chunks columns as [z][chunk][y][64] and a box of 64 columns, `rows` rows and 4 chunks.
template <typename T>
bool encode_rows(CUtensorMap* map, const void* base, int64_t x, int64_t y, int64_t z, int64_t y_stride, int64_t z_stride,
                 int rows, int64_t chunks = 0) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  // a dimension of one has no stride of its own, but the map wants one
  if (y == 1) y_stride = 64;
  if (z == 1) z_stride = 64;
  auto u = [](int64_t v) { return static_cast<cuuint64_t>(v); };
  const bool wide = chunks > 0;
  const cuuint64_t dims[4] = {u(wide ? 64 : x), u(y), u(wide ? chunks : z), u(z)};
  const cuuint64_t strides[3] = {u(y_stride * 2), u(wide ? 128 : z_stride * 2), u(z_stride * 2)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), wide ? 4u : 1u, 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                wide ? 4 : 3, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A kernel that may be set up while the one before it in the stream still runs (it waits for its end by
// itself, wait_for_previous_kernel).
template <typename K, typename... Args>
cudaError_t launch_dependent(K kernel, unsigned grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <typename T>
cudaError_t launch_attention(const PagedAttnArgs& a, const AttnPlan& plan, cudaStream_t stream) {
  CUtensorMap wide{}, runs, ql, qp;
  const int64_t width = a.latent + a.rope;
  if (!encode_rows<T>(&ql, a.q_latent, a.latent, a.heads, a.batch, a.ql_head_stride, a.ql_stride, kCtaHeads) ||
      !encode_rows<T>(&qp, a.q_pe, a.rope, a.heads, a.batch, a.qp_head_stride, a.qp_stride, kCtaHeads) ||
      !encode_rows<T>(&runs, a.cache, width, a.page_size, a.pages, a.row_stride, a.page_stride, plan.run) ||
      (plan.wide && !encode_rows<T>(&wide, a.cache, width, a.page_size, a.pages, a.row_stride, a.page_stride, plan.run, a.latent / 64)))
    return cudaErrorInvalidValue;
  auto kernel = paged_attention_kernel<T>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kAttnSmem));
  if (err != cudaSuccess) return err;
  kernel<<<static_cast<unsigned>(2 * plan.workers), kAttnThreads, kAttnSmem, stream>>>(wide, runs, ql, qp, a, plan);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (a.batch * a.heads >= 12 * gemv_grid_ctas())
    return launch_dependent(paged_attention_join_kernel<T, 4>, static_cast<unsigned>(a.batch * ceil_div(a.heads, 4)), kJoinThreads, stream, a, plan);
  return launch_dependent(paged_attention_join_kernel<T, 1>, static_cast<unsigned>(a.batch * a.heads), kJoinThreads, stream, a, plan);
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
