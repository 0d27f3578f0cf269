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
// shuffles.
#include "fp8_gemv.cuh"
#include "router.cuh"
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
// Two floats -> two e4m3 codes, a in the low byte.
MOE_D uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

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

// Eight columns of a row: 16-byte accesses when VEC (whole and aligned), else
// one element at a time, `n` of them present.
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
#pragma unroll
    for (int i = 0; i < 8 * static_cast<int>(sizeof(T)) / 16; ++i)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(f[i]);
  }
}

// The group's scale and this lane's eight codes; the sixteen lanes of a group
// are neighbours and all take part.
template <bool VEC>
MOE_D void codes8(const float (&y)[8], int n, uint8_t* codes, float* scale, bool first) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(y[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const float s = max_nan(amax, kTinyAmax) / kE4m3Max;
  const float inv = 1.0f / s;  // a code off by its neighbour only within 2 ulp of a rounding border
  if (n <= 0) return;
  const uint32_t lo = e4m3x2(y[0] * inv, y[1] * inv) | e4m3x2(y[2] * inv, y[3] * inv) << 16;
  const uint32_t hi = e4m3x2(y[4] * inv, y[5] * inv) | e4m3x2(y[6] * inv, y[7] * inv) << 16;
  if (VEC) {
    *reinterpret_cast<uint2*>(codes) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) codes[i] = static_cast<uint8_t>((i < 4 ? lo >> (8 * i) : hi >> (8 * (i - 4))) & 0xFFu);
  }
  if (first) *scale = s;
}

MOE_D int columns_from(int64_t c, int64_t cols) { return static_cast<int>(cols - c < 8 ? cols - c : 8); }

// A row per CTA and step; thread t holds columns 8 (t + i blockDim) .. + 7,
// i < V, as fp32 values of the stored type.
template <typename T, typename W, bool VEC, int V>
__global__ void __launch_bounds__(1024) rmsnorm_fp8_kernel(NormArgs a) {
  __shared__ float part[32];
  const int t = threadIdx.x, nt = blockDim.x, lane = t % kWarp, warp = t / kWarp;
  const int64_t groups = ceil_div(a.cols, 128);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + r * a.residual_stride : nullptr;
    float h[V][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t c = 8 * (t + static_cast<int64_t>(i) * nt);
      const int n = columns_from(c, a.cols);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
      if (n > 0) {
        load8<T, VEC>(x + c, n, h[i]);
        if (res) {
          float e[8];
          load8<T, VEC>(res + c, n, e);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[i][j] = widen<T>(from_float<T>(h[i][j] + e[j]));
          store8<T, VEC>(static_cast<T*>(a.residual_out) + r * a.cols + c, n, h[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    }
    ss = warp_sum(ss);
    __syncthreads();  // the previous row's sums have been read
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < nt / kWarp; ++i) total += part[i];
    const float inv = 1.0f / sqrtf(total / static_cast<float>(a.cols) + a.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t c = 8 * (t + static_cast<int64_t>(i) * nt);
      const int n = columns_from(c, a.cols);
      float y[8];
      if (n > 0) load8<W, VEC>(static_cast<const W*>(a.weight) + c, n, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = n > 0 ? h[i][j] * inv * y[j] : 0.0f;
      if (a.normed_out && n > 0) store8<T, VEC>(static_cast<T*>(a.normed_out) + r * a.cols + c, n, y);
      codes8<VEC>(y, n, a.codes + r * a.codes_stride + c, a.scales + r * groups + c / 128, c % 128 == 0);
    }
  }
}

// Sixteen lanes per (row, group); whole warps stay together for the shuffles.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(NormArgs a) {
  const int64_t groups = ceil_div(a.cols, 128), units = a.rows * groups;
  const int sub = threadIdx.x % 16;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (256 / 16);
  for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * (256 / 16); u0 < units; u0 += step) {
    const int64_t u = u0 + threadIdx.x / 16;
    const int64_t r = u / groups, g = u - r * groups, c = g * 128 + sub * 8;
    const int n = u < units ? columns_from(c, a.cols) : 0;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = 0.0f;
    if (n > 0) load8<T, VEC>(static_cast<const T*>(a.x) + r * a.x_stride + c, n, y);
    codes8<VEC>(y, n, a.codes + r * a.codes_stride + c, a.scales + u, sub == 0);
  }
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T, typename W, bool VEC>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t stream) {
  const int64_t vectors = ceil_div(a.cols, 8);
  const int v = vectors <= 1024 ? 1 : vectors <= 2048 ? 2 : 4;
  const int threads = static_cast<int>(ceil_div(ceil_div(vectors, v), 32) * 32);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, int64_t(gemv_grid_ctas()) * 8));
  if (v == 1) rmsnorm_fp8_kernel<T, W, VEC, 1><<<grid, threads, 0, stream>>>(a);
  else if (v == 2) rmsnorm_fp8_kernel<T, W, VEC, 2><<<grid, threads, 0, stream>>>(a);
  else rmsnorm_fp8_kernel<T, W, VEC, 4><<<grid, threads, 0, stream>>>(a);
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
  const int64_t units = a.rows * ceil_div(a.cols, 128);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(units, 16), int64_t(gemv_grid_ctas()) * 64));
  if (vec) quantize_rows_kernel<T, true><<<grid, 256, 0, stream>>>(a);
  else quantize_rows_kernel<T, false><<<grid, 256, 0, stream>>>(a);
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
