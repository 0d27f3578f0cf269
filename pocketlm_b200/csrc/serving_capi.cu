// extern "C" entry points of the batched operators in front of the MoE layer
// (include/moe_b200.h): argument checks, scratch planning, launches.
#include "../../include/moe_b200.h"
#include "common.cuh"
#include "plan.cuh"
#include "router.cuh"
#include "serving.cuh"
#include "status.cuh"

using namespace moe;

namespace {

bool is_type(int d) { return d == kDtypeF32 || d == kDtypeBF16 || d == kDtypeF16; }
bool is_16bit(int d) { return d == kDtypeBF16 || d == kDtypeF16; }

}  // namespace

extern "C" {

int moe_rmsnorm_fp8(const void* x, int64_t x_stride, int x_dtype, const void* residual, int64_t residual_stride,
                    const void* weight, int weight_dtype, int64_t rows, int64_t cols, float eps, uint8_t* codes,
                    int64_t codes_stride, float* scales, void* residual_out, void* normed_out, void* stream) {
  if (!x || !weight || !codes || !scales || (residual && !residual_out)) return fail(kNullPointer, "null pointer");
  if (rows < 0 || cols <= 0 || codes_stride < cols) return fail(kBadDims, "bad dimensions");
  if (!is_type(x_dtype) || (weight_dtype != x_dtype && weight_dtype != kDtypeF32))
    return fail(kUnsupported, "x is fp32, bf16 or fp16 and the weight of x's type or fp32");
  if (cols > kNormMaxCols) return fail(kUnsupported, "more than 32768 columns");
  if (rows == 0) return kOk;
  NormArgs a{};
  a.x = x; a.residual = residual; a.weight = weight; a.residual_out = residual_out; a.normed_out = normed_out;
  a.codes = codes; a.scales = scales; a.rows = rows; a.cols = cols; a.x_stride = x_stride;
  a.residual_stride = residual_stride; a.codes_stride = codes_stride; a.eps = eps;
  MOE_CUDA(launch_rmsnorm_fp8(a, x_dtype, weight_dtype, as_stream(stream)), "rmsnorm_fp8");
  return kOk;
}

int moe_fp8_quantize_rows(const void* x, int64_t x_stride, int x_dtype, int64_t rows, int64_t cols, uint8_t* codes,
                          int64_t codes_stride, float* scales, void* stream) {
  if (!x || !codes || !scales) return fail(kNullPointer, "null pointer");
  if (rows < 0 || cols <= 0 || codes_stride < cols) return fail(kBadDims, "bad dimensions");
  if (!is_type(x_dtype)) return fail(kUnsupported, "x is fp32, bf16 or fp16");
  if (cols > INT32_MAX / 2) return fail(kUnsupported, "dimension too large");
  if (rows == 0) return kOk;
  NormArgs a{};
  a.x = x; a.codes = codes; a.scales = scales; a.rows = rows; a.cols = cols; a.x_stride = x_stride;
  a.codes_stride = codes_stride;
  MOE_CUDA(launch_quantize_rows(a, x_dtype, as_stream(stream)), "fp8_quantize_rows");
  return kOk;
}

static int linear_supported(int64_t rows, int64_t out_rows, int64_t in_cols) {
  if (rows < 0 || out_rows <= 0 || in_cols <= 0) return fail(kBadDims, "bad dimensions");
  if (rows > INT32_MAX - 256 || out_rows > INT32_MAX - 256 || in_cols > INT32_MAX - 256)
    return fail(kUnsupported, "a dimension beyond 32 bits");
  return kOk;
}

int moe_fp8_block_linear_tile(int64_t rows, int64_t out_rows, int64_t in_cols) {
  const int code = linear_supported(rows, out_rows, in_cols);
  if (code != kOk || rows == 0) return code;
  const LinearTile t = fp8_linear_tile(rows, out_rows, in_cols);
  return t.tokens * 1000 + t.outs;
}

int moe_fp8_block_linear(const uint8_t* x_codes, int64_t x_stride, const float* x_scales, const uint8_t* fp8_weight,
                         int64_t weight_stride, const float* scale_inv, int64_t rows, int64_t out_rows,
                         int64_t in_cols, void* out, int out_dtype, void* stream) {
  if (!x_codes || !x_scales || !fp8_weight || !scale_inv || !out) return fail(kNullPointer, "null pointer");
  const int code = linear_supported(rows, out_rows, in_cols);
  if (code != kOk) return code;
  if (x_stride < in_cols || weight_stride < in_cols) return fail(kBadDims, "bad dimensions");
  if (!is_type(out_dtype)) return fail(kUnsupported, "the output is fp32, bf16 or fp16");
  if (((reinterpret_cast<uintptr_t>(x_codes) | reinterpret_cast<uintptr_t>(fp8_weight)) & 15u) || x_stride % 16 ||
      weight_stride % 16)
    return fail(kUnsupported, "code rows must start on 16-byte boundaries");
  if (rows == 0) return kOk;
  LinearArgs a{};
  a.x = x_codes; a.x_scales = x_scales; a.w = fp8_weight; a.w_scales = scale_inv; a.out = out;
  a.rows = rows; a.outs = out_rows; a.cols = in_cols; a.x_stride = x_stride; a.w_stride = weight_stride;
  MOE_CUDA(launch_fp8_linear(a, out_dtype, as_stream(stream)), "fp8_block_linear");
  return kOk;
}

int moe_paged_mla_append(const void* kv_rows, int64_t kv_stride, int kv_dtype, const void* kv_norm_weight,
                         int norm_dtype, const int64_t* slots, const int64_t* positions, const float* rope_cos,
                         const float* rope_sin, int64_t table_rows, void* cache, int cache_dtype, int64_t pages,
                         int64_t page_size, int64_t page_stride, int64_t row_stride, const void* q_pe,
                         int64_t q_stride, int64_t q_head_stride, int64_t heads, void* q_out, int64_t tokens,
                         int64_t kv_lora_rank, int64_t qk_rope_dim, float rms_eps, void* stream) {
  if (!kv_rows || !kv_norm_weight || !slots || !positions || !rope_cos || !rope_sin || !cache || (q_pe && !q_out))
    return fail(kNullPointer, "null pointer");
  if (tokens < 0 || kv_lora_rank <= 0 || qk_rope_dim <= 0 || qk_rope_dim % 2 || table_rows <= 0 || pages <= 0 ||
      page_size <= 0 || heads < 0 || (q_pe && heads == 0))
    return fail(kBadDims, "bad dimensions");
  if (!is_16bit(cache_dtype) || (kv_dtype != cache_dtype && kv_dtype != kDtypeF32) ||
      (norm_dtype != cache_dtype && norm_dtype != kDtypeF32))
    return fail(kUnsupported, "the cache is bf16 or fp16; rows and norm weight of the cache's type or fp32");
  if (kv_lora_rank > 1024 || qk_rope_dim > 1024 || heads > (1 << 20)) return fail(kUnsupported, "dimension too large");
  // (a dimension of one has no stride)
  const int64_t width = kv_lora_rank + qk_rope_dim;
  if ((pages > 1 && page_stride < width) || (page_size > 1 && row_stride < width))
    return fail(kUnsupported, "the cache's rows overlap");
  if (tokens == 0) return kOk;
  AppendArgs a{};
  a.kv = kv_rows; a.norm_w = kv_norm_weight; a.slots = slots; a.positions = positions; a.cos = rope_cos;
  a.sin = rope_sin; a.cache = cache; a.q = q_pe; a.q_out = q_out; a.tokens = tokens; a.latent = kv_lora_rank;
  a.rope = qk_rope_dim; a.heads = heads; a.kv_stride = kv_stride; a.q_stride = q_stride;
  a.q_head_stride = q_head_stride; a.pages = pages; a.page_size = page_size; a.page_stride = page_stride;
  a.row_stride = row_stride; a.table_rows = table_rows; a.eps = rms_eps;
  MOE_CUDA(launch_paged_append(a, kv_dtype, norm_dtype, cache_dtype, as_stream(stream)), "paged_mla_append");
  return kOk;
}

static int attention_supported(int64_t batch, int64_t heads, int64_t latent, int64_t rope, int64_t table_cols,
                               int64_t page_size) {
  if (batch < 0 || heads <= 0 || latent <= 0 || rope <= 0 || table_cols <= 0 || page_size <= 0)
    return fail(kBadDims, "bad dimensions");
  if (latent > 512 || latent % 8 || rope > 64 || rope % 8)
    return fail(kUnsupported, "kv_lora_rank up to 512 and qk_rope_dim up to 64, multiples of 8");
  // (positions, rounded up to whole tiles, stay inside 32 bits)
  if (batch > 65535 || heads > (1 << 16) || batch * heads > INT32_MAX || table_cols > (INT32_MAX - 256) / page_size)
    return fail(kUnsupported, "dimension too large");
  return kOk;
}

int64_t moe_paged_mla_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_lora_rank,
                                                int64_t qk_rope_dim, int64_t table_cols, int64_t page_size) {
  if (attention_supported(batch, heads, kv_lora_rank, qk_rope_dim, table_cols, page_size) != kOk) return -1;
  return paged_attn_workspace_bytes(batch, heads, kv_lora_rank, table_cols, page_size);
}

int moe_paged_mla_attention(const void* q_latent, int64_t ql_stride, int64_t ql_head_stride, const void* q_pe,
                            int64_t qp_stride, int64_t qp_head_stride, const void* cache, int dtype, int64_t pages,
                            int64_t page_size, int64_t page_stride, int64_t row_stride, const int32_t* page_table,
                            int64_t table_stride, int64_t table_cols, const int32_t* lengths, int64_t batch,
                            int64_t heads, int64_t kv_lora_rank, int64_t qk_rope_dim, float softmax_scale, void* out,
                            float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q_latent || !q_pe || !cache || !page_table || !lengths || !out) return fail(kNullPointer, "null pointer");
  const int code = attention_supported(batch, heads, kv_lora_rank, qk_rope_dim, table_cols, page_size);
  if (code != kOk) return code;
  if (pages <= 0) return fail(kBadDims, "bad dimensions");
  if (pages >= INT32_MAX) return fail(kUnsupported, "dimension too large");
  if (!is_16bit(dtype)) return fail(kUnsupported, "queries and cache are bf16 or fp16");
  if (!(softmax_scale >= 0.0f) || softmax_scale > 3.0e38f) return fail(kBadDims, "softmax_scale must be finite and not negative");
  if (((reinterpret_cast<uintptr_t>(q_latent) | reinterpret_cast<uintptr_t>(q_pe) | reinterpret_cast<uintptr_t>(cache) |
        reinterpret_cast<uintptr_t>(out)) & 15u) ||
      (ql_stride | ql_head_stride | qp_stride | qp_head_stride | page_stride | row_stride) % 8)
    return fail(kUnsupported, "rows of queries and cache must start on 16-byte boundaries");
  // (a dimension of one has no stride)
  if ((batch > 1 && (ql_stride <= 0 || qp_stride <= 0)) || (heads > 1 && (ql_head_stride <= 0 || qp_head_stride <= 0)) ||
      (pages > 1 && page_stride <= 0) || (page_size > 1 && row_stride <= 0))
    return fail(kUnsupported, "strides must be positive");
  if (reinterpret_cast<uintptr_t>(workspace) & 31u) return fail(kUnsupported, "the workspace must start on a 32-byte boundary");
  if (batch == 0) return kOk;
  PagedAttnArgs a{};
  a.q_latent = q_latent; a.q_pe = q_pe; a.cache = cache; a.table = page_table; a.lengths = lengths; a.out = out;
  a.lse = lse; a.batch = batch; a.heads = heads; a.latent = kv_lora_rank; a.rope = qk_rope_dim;
  a.ql_stride = ql_stride; a.ql_head_stride = ql_head_stride; a.qp_stride = qp_stride;
  a.qp_head_stride = qp_head_stride; a.pages = pages; a.page_size = page_size; a.page_stride = page_stride;
  a.row_stride = row_stride; a.table_cols = table_cols; a.table_stride = table_stride; a.scale = softmax_scale;
  cudaStream_t s = as_stream(stream);
  const int64_t need = paged_attn_workspace_bytes(batch, heads, kv_lora_rank, table_cols, page_size);
  Scratch scratch(workspace, workspace_bytes, static_cast<size_t>(need), s);
  if (!scratch.ok()) return fail(kNoMemory, "workspace too small or allocation failed");
  MOE_CUDA(launch_paged_attention(a, dtype, scratch.base(), s), "paged_mla_attention");
  return kOk;
}

}  // extern "C"
