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
#include "serving.cuh"

namespace moe {
namespace {

template <typename T>
MOE_D T from_float(float v);
template <>
MOE_D float from_float<float>(float v) { return v; }
template <>
MOE_D __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
MOE_D __half from_float<__half>(float v) { return __float2half_rn(v); }
template <typename T>
MOE_D float widen(T v) { return static_cast<float>(v); }

// Eight values: 16-byte accesses when VEC, else the first n one at a time.
template <typename T, bool VEC>
MOE_D void load8(const T* p, int n, float (&f)[8]) {
  if (VEC) {
    constexpr int kV = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / kV; ++i) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p) + i), f + i * kV);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? widen<T>(p[i]) : 0.0f;
  }
}
template <typename T, bool VEC>
MOE_D void store8(T* p, int n, const float (&f)[8]) {
  if (VEC) {
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_float<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(f[i]);
  }
}

constexpr int kAppendThreads = 256;
constexpr int kAppendVectors = 4;  // 8-value vectors of a latent row per lane: latent <= 1024

// Pairs (2p, 2p + 1) of eight values from column c of a rope group, turned.
MOE_D void rotate8(float (&f)[8], int n, const float* cos, const float* sin, int64_t c) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    if (2 * p >= n) break;
    const float cs = __ldg(cos + c / 2 + p), sn = __ldg(sin + c / 2 + p);
    const float a = f[2 * p], b = f[2 * p + 1];
    f[2 * p] = a * cs - b * sn;
    f[2 * p + 1] = a * sn + b * cs;
  }
}

// Unit u of a token: 0 its cache row, 1 .. its queries' rope values 256 (u - 1) .. + 255.
template <typename T, typename W, typename C, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(AppendArgs a, int units) {
  const int lane = threadIdx.x % kWarp;
  const int64_t total = a.tokens * units, warps = static_cast<int64_t>(gridDim.x) * (kAppendThreads / kWarp);
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x) / kWarp; i < total; i += warps) {
    const int64_t t = i / units;
    const int unit = static_cast<int>(i - t * units);
    const int64_t slot = a.slots[t], pos = a.positions[t];
    const bool placed = pos >= 0 && pos < a.table_rows;
    const float* cos = a.cos + (placed ? pos : 0) * (a.rope / 2);
    const float* sin = a.sin + (placed ? pos : 0) * (a.rope / 2);
    if (unit == 0) {
      if (slot < 0) continue;
      if (!placed || slot >= a.pages * a.page_size) {
        if (lane == 0) atomicOr(&g_device_error, kPagedRangeError);
        continue;
      }
      const T* src = static_cast<const T*>(a.kv) + t * a.kv_stride;
      const int64_t page = slot / a.page_size;
      C* dst = static_cast<C*>(a.cache) + page * a.page_stride + (slot - page * a.page_size) * a.row_stride;
      float f[kAppendVectors][8];
      float ss = 0.0f;
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v) {
        const int64_t c = 8 * (lane + static_cast<int64_t>(v) * kWarp);
        const int n = static_cast<int>(a.latent - c < 8 ? a.latent - c : 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[v][j] = 0.0f;
        if (n > 0) load8<T, VEC>(src + c, n, f[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(f[v][j], f[v][j], ss);
      }
      const float inv = 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(a.latent) + a.eps);
#pragma unroll
      for (int v = 0; v < kAppendVectors; ++v) {
        const int64_t c = 8 * (lane + static_cast<int64_t>(v) * kWarp);
        const int n = static_cast<int>(a.latent - c < 8 ? a.latent - c : 8);
        if (n <= 0) continue;
        float w[8];
        load8<W, VEC>(static_cast<const W*>(a.norm_w) + c, n, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[v][j] *= inv * w[j];
        store8<C, VEC>(dst + c, n, f[v]);
      }
      for (int64_t c = 8 * lane; c < a.rope; c += 8 * kWarp) {
        const int n = static_cast<int>(a.rope - c < 8 ? a.rope - c : 8);
        load8<T, VEC>(src + a.latent + c, n, f[0]);
        rotate8(f[0], n, cos, sin, c);
        store8<C, VEC>(dst + a.latent + c, n, f[0]);
      }
    } else {
      // eight values of one head's group per lane (groups of eight never cross heads)
      const int64_t per_head = ceil_div(a.rope, 8);
      const int64_t v = (unit - 1) * static_cast<int64_t>(kWarp) + lane, h = v / per_head;
      if (h >= a.heads) continue;
      const int64_t c = 8 * (v - h * per_head);
      const int n = static_cast<int>(a.rope - c < 8 ? a.rope - c : 8);
      float f[8];
      load8<C, VEC>(static_cast<const C*>(a.q) + t * a.q_stride + h * a.q_head_stride + c, n, f);
      if (placed) {
        rotate8(f, n, cos, sin, c);
      } else {  // a row that has no place in the sequence: zeros
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.0f;
      }
      store8<C, VEC>(static_cast<C*>(a.q_out) + (t * a.heads + h) * a.rope + c, n, f);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, typename W, typename C>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
  const int64_t units = 1 + (a.q ? ceil_div(a.heads * ceil_div(a.rope, 8), kWarp) : 0);
  auto whole = [](int64_t n, int64_t size) { return n * size % 16 == 0; };
  const bool vec = a.latent % 8 == 0 && a.rope % 8 == 0 && aligned16(a.kv) && whole(a.kv_stride, sizeof(T)) &&
                   aligned16(a.norm_w) && aligned16(a.cache) && whole(a.page_stride, sizeof(C)) &&
                   whole(a.row_stride, sizeof(C)) &&
                   (!a.q || (aligned16(a.q) && aligned16(a.q_out) && whole(a.q_stride, sizeof(C)) &&
                             whole(a.q_head_stride, sizeof(C))));
  const int64_t ctas = ceil_div(a.tokens * units, kAppendThreads / kWarp);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ctas, int64_t(gemv_grid_ctas()) * 32));
  if (vec) paged_append_kernel<T, W, C, true><<<grid, kAppendThreads, 0, stream>>>(a, static_cast<int>(units));
  else paged_append_kernel<T, W, C, false><<<grid, kAppendThreads, 0, stream>>>(a, static_cast<int>(units));
  return cudaGetLastError();
}

template <typename C>
cudaError_t launch_append_types(const AppendArgs& a, int x_dtype, int norm_dtype, cudaStream_t stream) {
  const bool wide = norm_dtype == kDtypeF32;
  if (x_dtype == kDtypeF32)
    return wide ? launch_append<float, float, C>(a, stream) : launch_append<float, C, C>(a, stream);
  return wide ? launch_append<C, float, C>(a, stream) : launch_append<C, C, C>(a, stream);
}

// One CTA per (row, head): its warps take positions in turn, each with a
// running maximum, sum and latent sums, joined at the end.
constexpr int kSimpleWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * kWarp) paged_attention_simple_kernel(PagedAttnArgs a) {
  constexpr int kCols = 16;  // latent columns per lane: latent <= 512
  __shared__ float m_s[kSimpleWarps], l_s[kSimpleWarps], acc_s[kSimpleWarps][kCols * kWarp];
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int64_t b = blockIdx.y, h = blockIdx.x;
  const T* ql = static_cast<const T*>(a.q_latent) + b * a.ql_stride + h * a.ql_head_stride;
  const T* qp = static_cast<const T*>(a.q_pe) + b * a.qp_stride + h * a.qp_head_stride;
  const int64_t len = std::max(0, a.lengths[b]);
  float acc[kCols];
  for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  for (int64_t p = warp; p < len; p += kSimpleWarps) {
    const int64_t col = p / a.page_size;
    const int64_t page = col < a.table_cols ? a.table[b * a.table_stride + col] : -1;
    if (page < 0 || page >= a.pages) {
      if (lane == 0) atomicOr(&g_device_error, kPagedRangeError);
      continue;
    }
    const T* row = static_cast<const T*>(a.cache) + page * a.page_stride + (p - col * a.page_size) * a.row_stride;
    float s = 0.0f, c[kCols];
    for (int i = 0; i < kCols; ++i) {
      const int k = lane + i * kWarp;
      c[i] = k < a.latent ? widen<T>(row[k]) : 0.0f;
      if (k < a.latent) s = fmaf(widen<T>(ql[k]), c[i], s);
    }
    for (int k = lane; k < a.rope; k += kWarp) s = fmaf(widen<T>(qp[k]), widen<T>(row[a.latent + k]), s);
    s = warp_sum(s) * a.scale;
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.0f : expf(m - top), e = expf(s - top);
    l = l * old + e;
    for (int i = 0; i < kCols; ++i) acc[i] = acc[i] * old + e * c[i];
    m = top;
  }
  for (int i = 0; i < kCols; ++i) acc_s[warp][lane + i * kWarp] = acc[i];
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.0f;
  for (int w = 0; w < kSimpleWarps; ++w) top = fmaxf(top, m_s[w]);
  for (int w = 0; w < kSimpleWarps; ++w) total += l_s[w] == 0.0f ? 0.0f : l_s[w] * expf(m_s[w] - top);
  for (int k = threadIdx.x; k < a.latent; k += kSimpleWarps * kWarp) {
    float v = 0.0f;
    for (int w = 0; w < kSimpleWarps; ++w)
      if (l_s[w] != 0.0f) v += acc_s[w][k] * expf(m_s[w] - top);
    static_cast<T*>(a.out)[(b * a.heads + h) * a.latent + k] = from_float<T>(total == 0.0f ? 0.0f : v / total);
  }
  if (a.lse && threadIdx.x == 0) a.lse[b * a.heads + h] = total == 0.0f ? -INFINITY : top + logf(total);
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs& a, int x_dtype, int norm_dtype, int cache_dtype, cudaStream_t stream) {
  if (cache_dtype == kDtypeBF16) return launch_append_types<__nv_bfloat16>(a, x_dtype, norm_dtype, stream);
  return launch_append_types<__half>(a, x_dtype, norm_dtype, stream);
}

int64_t paged_attn_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, char*, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.heads), static_cast<unsigned>(a.batch));
  if (dtype == kDtypeBF16) paged_attention_simple_kernel<__nv_bfloat16><<<grid, kSimpleWarps * kWarp, 0, stream>>>(a);
  else paged_attention_simple_kernel<__half><<<grid, kSimpleWarps * kWarp, 0, stream>>>(a);
  return cudaGetLastError();
}

int read_and_clear_paged_error(cudaStream_t stream) { return read_and_clear_local_error(stream); }

}  // namespace moe
