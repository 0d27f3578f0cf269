// The batched operators in front of the MoE layer (8-bit RMSNorm rows, the
// block-scaled FP8 linear, the paged latent cache and its attention): the
// arguments their kernels take.  Strides are in elements.
#pragma once
#include "common.cuh"

namespace moe {

// moe_b200_device_error codes of these operators
constexpr int kPagedRangeError = 512;   // a slot, position, page or length outside its range: skipped
constexpr int kLinearWaitError = 1024;  // a bounded wait of the FP8 linear ran out
constexpr int kPagedWaitError = 2048;   // a bounded wait of the paged attention ran out

// ---- norm_fp8.cu
struct NormArgs {
  const void* x;         // [rows, cols], rows x_stride apart
  const void* residual;  // added when given
  const void* weight;    // [cols]
  void* residual_out;    // [rows, cols]: x + residual in x's type (with residual)
  void* normed_out;      // [rows, cols] in x's type, or null
  uint8_t* codes;        // [rows, cols], rows codes_stride apart
  float* scales;         // [rows, ceil(cols / 128)]
  int64_t rows, cols, x_stride, residual_stride, codes_stride;
  float eps;
};
constexpr int64_t kNormMaxCols = 32768;
cudaError_t launch_rmsnorm_fp8(const NormArgs& a, int x_dtype, int weight_dtype, cudaStream_t stream);
cudaError_t launch_quantize_rows(const NormArgs& a, int x_dtype, cudaStream_t stream);

// ---- fp8_linear_tc.cu
struct LinearArgs {
  const uint8_t* x;       // [rows, cols] e4m3, rows x_stride apart
  const float* x_scales;  // [rows, kblocks]
  const uint8_t* w;       // [outs, cols] e4m3, rows w_stride apart
  const float* w_scales;  // [ceil(outs / 128), kblocks]
  void* out;              // [rows, outs]
  int64_t rows, outs, cols, x_stride, w_stride;
};
// The kernel that a call takes: weight streaming with 128 outputs and 16 to 128 tokens per CTA, or tiles of
// 192 to 256 outputs and 256 tokens (a pair of CTAs) or 128 (one).
struct LinearTile {
  int tokens, outs;
};
LinearTile fp8_linear_tile(int64_t rows, int64_t outs, int64_t cols);
cudaError_t launch_fp8_linear(const LinearArgs& a, int out_dtype, cudaStream_t stream);
int read_and_clear_linear_error(cudaStream_t stream);

// ---- paged_mla.cu
struct AppendArgs {
  const void* kv;         // [tokens, latent + rope], rows kv_stride apart
  const void* norm_w;     // [latent]
  const int64_t* slots;   // [tokens]: page * page_size + offset, negative = no row to store
  const int64_t* positions;
  const float* cos;       // [table_rows, rope / 2]
  const float* sin;
  void* cache;            // [pages, page_size, latent + rope]
  const void* q;          // [tokens, heads, rope] or null
  void* q_out;            // [tokens, heads, rope], contiguous
  int64_t tokens, latent, rope, heads, kv_stride, q_stride, q_head_stride;
  int64_t pages, page_size, page_stride, row_stride, table_rows;
  float eps;
};
cudaError_t launch_paged_append(const AppendArgs& a, int x_dtype, int norm_dtype, int cache_dtype, cudaStream_t stream);

struct PagedAttnArgs {
  const void* q_latent;  // [batch, heads, latent]
  const void* q_pe;      // [batch, heads, rope]
  const void* cache;     // [pages, page_size, latent + rope]
  const int32_t* table;  // [batch, table_cols]
  const int32_t* lengths;
  void* out;             // [batch, heads, latent], contiguous
  float* lse;            // [batch, heads] or null
  int64_t batch, heads, latent, rope;
  int64_t ql_stride, ql_head_stride, qp_stride, qp_head_stride;
  int64_t pages, page_size, page_stride, row_stride, table_cols, table_stride;
  float scale;
};
int64_t paged_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t latent, int64_t table_cols, int64_t page_size);
cudaError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, char* workspace, cudaStream_t stream);
int read_and_clear_paged_error(cudaStream_t stream);

}  // namespace moe
