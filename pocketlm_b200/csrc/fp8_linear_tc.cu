// The block-scaled FP8 linear for batches whose rows are e4m3 too:
//   out[t, n] = sum_g sx[t, g] sw[n / 128, g] sum_{k in group g} x[t, k] w[n, k],
// groups of 128 columns, 128 x 128 weight blocks; products and sums in fp32,
// one rounding to the output's type.
#include <algorithm>

#include "async_copy.cuh"
#include "fp8_gemv.cuh"
#include "router.cuh"
#include "serving.cuh"

namespace moe {
namespace {

// A 64 x 64 tile of the output per CTA, 16 columns of k a step.
constexpr int kT = 64, kK = 16;
template <typename O>
__global__ void __launch_bounds__(256) fp8_linear_simple_kernel(LinearArgs a) {
  __shared__ float xs[kK][kT + 4], ws[kK][kT + 4];
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * kT, n0 = static_cast<int64_t>(blockIdx.x) * kT;
  const int64_t kb = ceil_div(a.cols, 128);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < a.cols; k0 += kK) {
    for (int i = threadIdx.x; i < kT * kK; i += 256) {
      const int r = i / kK, c = i % kK;
      const int64_t k = k0 + c, t = t0 + r, n = n0 + r;
      xs[c][r] = t < a.rows && k < a.cols ? e4m3x2_to_float2(a.x[t * a.x_stride + k]).x * a.x_scales[t * kb + k / 128] : 0.0f;
      ws[c][r] = n < a.outs && k < a.cols ? e4m3x2_to_float2(a.w[n * a.w_stride + k]).x * a.w_scales[n / 128 * kb + k / 128] : 0.0f;
    }
    __syncthreads();
    for (int c = 0; c < kK; ++c)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[c][ty * 4 + i], ws[c][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t t = t0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (t < a.rows && n < a.outs) static_cast<O*>(a.out)[t * a.outs + n] = static_cast<O>(acc[i][j]);
    }
}

}  // namespace

cudaError_t launch_fp8_linear(const LinearArgs& a, int out_dtype, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.outs, kT)), static_cast<unsigned>(ceil_div(a.rows, kT)));
  if (out_dtype == kDtypeF32) fp8_linear_simple_kernel<float><<<grid, 256, 0, stream>>>(a);
  else if (out_dtype == kDtypeBF16) fp8_linear_simple_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else fp8_linear_simple_kernel<__half><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError();
}

int read_and_clear_linear_error(cudaStream_t stream) { return read_and_clear_local_error(stream); }

}  // namespace moe
