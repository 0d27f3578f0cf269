// RMSNorm with the residual's addition and an 8-bit output, and the same
// 8-bit form of rows without a norm:
//   h = round(x + residual)                      (the stream, kept in x's type)
//   y = h / sqrt(mean(h^2) + eps) * w            (fp32)
//   scale[g] = max(amax of y over columns 128 g .. 128 g + 127, 2^-100) / 448
//   code = e4m3(y / scale[g])                    (to nearest even, saturating)
// The mean is of the stream as it is stored, so a later layer that reads the
// stream sees the values that were normalised here.  The floor under the amax
// gives an all-zero group a finite scale and zero codes.  A NaN in a group
// makes its scale and codes NaN (max.NaN below); an infinity makes its
// scale infinite, its own code NaN and the group's other codes zero.
//
// Bytes bound both (a row is read once and kept in registers between the
// mean and the codes).  Eight consecutive columns belong to a thread, so
// sixteen neighbouring lanes hold a scale group and find its amax with four
// shuffles.  Measured, bf16, inputs from memory, 1965 MHz: 8192 x 7168 with the
// residual and the 16-bit rows 89 us (530 MB, 5.9 TB/s), one row 3.4 us (2.8 from
// L2); 4096 x 16384 without a norm 36 us (203 MB, 5.7 TB/s), 64 x 16384 3.2 us.
// Where columns, a pointer or a row stride do not allow 16-byte accesses, every
// array goes element by element: with rows of x one value longer the first takes
// 390 us, 4096 x 16384 134 us.
#include <algorithm>

#include "fp8_gemv.cuh"
#include "router.cuh"
#include "rows.cuh"
#include "serving.cuh"

namespace moe {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kTinyAmax = 7.888609052210118e-31f;  // 2^-100

MOE_D float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
MOE_D float reciprocal(float a) {  // within 1 ulp; 0 of an infinity
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
// Two floats -> two e4m3 codes, a in the low byte.
MOE_D uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

MOE_D int columns_from(int64_t c, int64_t cols) { return static_cast<int>(cols - c < 8 ? cols - c : 8); }

// The largest size among eight stored values (NaN if one is).
template <typename T>
MOE_D float amax8(const Eight<T>& e) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(widen<T>(e.v[i])));
  return m;
}
template <>
MOE_D float amax8<__nv_bfloat16>(const Eight<__nv_bfloat16>& e) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(e.v);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
  return max_nan(__low2float(m), __high2float(m));
}
template <>
MOE_D float amax8<__half>(const Eight<__half>& e) {
  const __half2* p = reinterpret_cast<const __half2*>(e.v);
  const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
  return max_nan(__low2float(m), __high2float(m));
}

// A group's scale and what codes are made with: y / s as the product with the
// reciprocal and one Newton step on its remainder, so that a value on the border
// between two codes goes to the even one (an infinite scale has no remainder: 0 * inf).
struct Scale {
  float s, inv, rem;
};
MOE_D Scale scale_of(float amax) {
  // amax / 448 and its reciprocal: an approximation and one Newton step each are enough
  amax = max_nan(amax, kTinyAmax);
  const float p = amax * (1.0f / kE4m3Max);
  Scale r;
  r.s = p > kE4m3Max * 1e30f ? p : fmaf(fmaf(-p, kE4m3Max, amax), 1.0f / kE4m3Max, p);
  r.inv = reciprocal(r.s);
  r.rem = r.inv == 0.0f ? 0.0f : -r.s;
  return r;
}
MOE_D uint32_t two_codes(float2 y, const Scale& s) {
  const float2 p = mul2(y, make_float2(s.inv, s.inv));
  const float2 q = fma2(fma2(p, make_float2(s.rem, s.rem), y), make_float2(s.inv, s.inv), p);
  return e4m3x2(q.x, q.y);
}
// Eight codes: 8 bytes at once when VEC, else the first n one at a time.
template <bool VEC>
MOE_D void store_codes8(uint8_t* codes, uint32_t lo, uint32_t hi, int n) {
  if (VEC) {
    *reinterpret_cast<uint2*>(codes) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) codes[i] = static_cast<uint8_t>((i < 4 ? lo >> (8 * i) : hi >> (8 * (i - 4))) & 0xFFu);
  }
}

// The group's scale and this lane's eight codes; the sixteen lanes of a group
// are neighbours and all take part.
template <bool VEC>
MOE_D void codes8(const float2 (&y)[4], float amax, int n, uint8_t* codes, float* scale, bool first) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const Scale s = scale_of(amax);
  if (n <= 0) return;
  store_codes8<VEC>(codes, two_codes(y[0], s) | two_codes(y[1], s) << 16, two_codes(y[2], s) | two_codes(y[3], s) << 16, n);
  if (first) *scale = s.s;
}

// A row per CTA and step; thread t holds columns 8 (t + i blockDim) .. + 7,
// i < V, in the stored type.  All loads of a row are in flight before the first
// is used; many narrow CTAs per SM overlap one row's sum with others' bytes.
template <typename T, typename W, bool VEC, int V>
__global__ void __launch_bounds__(V == 1 ? 1024 : 512, V == 4 ? 2 : 1) rmsnorm_fp8_kernel(NormArgs a) {
  __shared__ float part[2][32];
  const int t = threadIdx.x, nt = blockDim.x, lane = t % kWarp, warp = t / kWarp;
  const int64_t groups = ceil_div(a.cols, 128);
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    Eight<T> h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = 8 * (t + i * nt), n = columns_from(c, a.cols);
      clear8(h[i]);
      if (n > 0) load8<T, VEC>(x + c, n, h[i]);
    }
    if (a.residual) {
      const T* res = static_cast<const T*>(a.residual) + r * a.residual_stride;
      Eight<T> e[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = 8 * (t + i * nt), n = columns_from(c, a.cols);
        clear8(e[i]);
        if (n > 0) load8<T, VEC>(res + c, n, e[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = 8 * (t + i * nt), n = columns_from(c, a.cols);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i].v[j] = from_float<T>(widen<T>(h[i].v[j]) + widen<T>(e[i].v[j]));
        if (n > 0) store8<T, VEC>(static_cast<T*>(a.residual_out) + r * a.cols + c, n, h[i]);
      }
    }
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(widen<T>(h[i].v[j]), widen<T>(h[i].v[j]), ss);
    ss = warp_sum(ss);
    if (lane == 0) part[turn][warp] = ss;
    __syncthreads();  // one per row: the other half of `part` is written meanwhile
    float total = 0.0f;
    for (int i = 0; i < nt / kWarp; ++i) total += part[turn][i];
    const float inv = 1.0f / sqrtf(total / static_cast<float>(a.cols) + a.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = 8 * (t + i * nt), n = columns_from(c, a.cols);
      if (V > 1 && c - 8 * lane >= a.cols) break;  // the whole warp is past the row
      Eight<W> w;
      clear8(w);
      if (n > 0) load8<W, VEC>(static_cast<const W*>(a.weight) + c, n, w);
      float2 y[4];
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j].x = n > 0 ? widen<T>(h[i].v[2 * j]) * inv * widen<W>(w.v[2 * j]) : 0.0f;
        y[j].y = n > 0 ? widen<T>(h[i].v[2 * j + 1]) * inv * widen<W>(w.v[2 * j + 1]) : 0.0f;
        amax = max_nan(amax, max_nan(fabsf(y[j].x), fabsf(y[j].y)));
      }
      if (a.normed_out && n > 0) {
        Eight<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = from_float<T>(j % 2 ? y[j / 2].y : y[j / 2].x);
        store8<T, VEC>(static_cast<T*>(a.normed_out) + r * a.cols + c, n, o);
      }
      codes8<VEC>(y, amax, n, a.codes + r * a.codes_stride + c, a.scales + r * groups + c / 128, c % 128 == 0);
    }
  }
}

// Eight lanes per (row, group), sixteen columns each, and kUnits groups per lane
// with their loads in flight together; whole warps stay together for the
// shuffles.  (With sixteen lanes of eight columns the shuffles and scales, done by
// every lane, kept the issue slots 77 % busy: 49 us on 4096 x 16384.)
constexpr int kUnits = 2, kQuantThreads = 256, kCtaUnits = kQuantThreads / 8 * kUnits;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(NormArgs a) {
  const int64_t groups = ceil_div(a.cols, 128), units = a.rows * groups;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kCtaUnits;
  const int64_t row0 = units <= UINT32_MAX ? static_cast<uint32_t>(first) / static_cast<uint32_t>(groups) : first / groups;
  const uint32_t rest = static_cast<uint32_t>(first - row0 * groups), per_row = static_cast<uint32_t>(groups);
  const int sub = threadIdx.x % 8;
  Eight<T> e[kUnits][2];
  int64_t row[kUnits];
  int col[kUnits], n[kUnits][2];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const uint32_t local = rest + threadIdx.x / 8 + i * (kQuantThreads / 8), r = local / per_row;
    row[i] = row0 + r;
    col[i] = static_cast<int>(local - r * per_row) * 128 + sub * 16;
    const bool in = first + threadIdx.x / 8 + i * (kQuantThreads / 8) < units;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      n[i][k] = in ? columns_from(col[i] + 8 * k, a.cols) : 0;
      clear8(e[i][k]);
      if (n[i][k] > 0) load8<T, VEC>(static_cast<const T*>(a.x) + row[i] * a.x_stride + col[i] + 8 * k, n[i][k], e[i][k]);
    }
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    float amax = max_nan(amax8<T>(e[i][0]), amax8<T>(e[i][1]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const Scale s = scale_of(amax);
    if (n[i][0] <= 0) continue;
    uint32_t c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const T* v = e[i][k / 2].v + 4 * (k % 2);
      c[k] = two_codes(make_float2(widen<T>(v[0]), widen<T>(v[1])), s) | two_codes(make_float2(widen<T>(v[2]), widen<T>(v[3])), s) << 16;
    }
    uint8_t* codes = a.codes + row[i] * a.codes_stride + col[i];
    store_codes8<VEC>(codes, c[0], c[1], n[i][0]);
    if (n[i][1] > 0) store_codes8<VEC>(codes + 8, c[2], c[3], n[i][1]);
    if (sub == 0) a.scales[row[i] * groups + col[i] / 128] = s.s;
  }
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, typename W, bool VEC>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t stream) {
  // No more rows than SMs: a thread per vector, the shortest way through a row
  // (7168 columns, inputs in L2, 1 row 3.1 us against 4.3, 148 rows 3.3 against
  // 4.6).  More: four vectors per thread, more rows at once (296 rows 5.3 us
  // against 5.7, 592 8.8 against 12.6).
  const int64_t vectors = ceil_div(a.cols, 8);
  const int v = vectors <= 1024 && a.rows <= gemv_grid_ctas() ? 1 : vectors <= 2048 ? 4 : 8;
  const int threads = static_cast<int>(ceil_div(ceil_div(vectors, v), 32) * 32);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, INT32_MAX));
  if (v == 1) rmsnorm_fp8_kernel<T, W, VEC, 1><<<grid, threads, 0, stream>>>(a);
  else if (v == 4) rmsnorm_fp8_kernel<T, W, VEC, 4><<<grid, threads, 0, stream>>>(a);
  else rmsnorm_fp8_kernel<T, W, VEC, 8><<<grid, threads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename W>
cudaError_t launch_norm_vec(const NormArgs& a, cudaStream_t stream) {
  const int64_t s = sizeof(T);
  const bool vec = a.cols % 8 == 0 && aligned(a.x, 16) && a.x_stride * s % 16 == 0 && aligned(a.weight, 16) &&
                   aligned(a.codes, 8) && a.codes_stride % 8 == 0 &&
                   (!a.residual || (aligned(a.residual, 16) && a.residual_stride * s % 16 == 0 && aligned(a.residual_out, 16))) &&
                   aligned(a.normed_out, 16);
  return vec ? launch_norm<T, W, true>(a, stream) : launch_norm<T, W, false>(a, stream);
}

template <typename T>
cudaError_t launch_norm_weight(const NormArgs& a, int weight_dtype, cudaStream_t stream) {
  if (weight_dtype == kDtypeF32) return launch_norm_vec<T, float>(a, stream);
  return launch_norm_vec<T, T>(a, stream);
}

template <typename T>
cudaError_t launch_quant(const NormArgs& a, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned(a.x, 16) && a.x_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                   aligned(a.codes, 8) && a.codes_stride % 8 == 0;
  const int64_t ctas = ceil_div(a.rows * ceil_div(a.cols, 128), kCtaUnits);
  if (ctas > INT32_MAX || a.cols > INT32_MAX / 2) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (vec) quantize_rows_kernel<T, true><<<grid, kQuantThreads, 0, stream>>>(a);
  else quantize_rows_kernel<T, false><<<grid, kQuantThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rmsnorm_fp8(const NormArgs& a, int x_dtype, int weight_dtype, cudaStream_t stream) {
  switch (x_dtype) {
    case kDtypeF32: return launch_norm_weight<float>(a, weight_dtype, stream);
    case kDtypeBF16: return launch_norm_weight<__nv_bfloat16>(a, weight_dtype, stream);
    default: return launch_norm_weight<__half>(a, weight_dtype, stream);
  }
}

cudaError_t launch_quantize_rows(const NormArgs& a, int x_dtype, cudaStream_t stream) {
  switch (x_dtype) {
    case kDtypeF32: return launch_quant<float>(a, stream);
    case kDtypeBF16: return launch_quant<__nv_bfloat16>(a, stream);
    default: return launch_quant<__half>(a, stream);
  }
}

}  // namespace moe
