"""Batched operators in front of the MoE layer, for serving many sequences.

The reference's attention block (native/__init__.py:878-1075) takes one fp32
token and a contiguous cache; these are its steps for a batch of tokens in
16 bits, 8-bit linears and a paged cache:

  rmsnorm_fp8          the residual's addition, RMSNorm, e4m3 rows with a scale per 128 columns
  quantize_fp8_rows    the same 8-bit form of rows as they are
  fp8_block_linear     e4m3 rows times an e4m3 weight with 128 x 128 block scales
  paged_mla_append     a batch's new latent rows into a paged cache, positions rotated on the way
  paged_mla_attention  one query token per row over its pages

Every tensor is on one CUDA device, which need not be the current one; the
work is enqueued on that device's current stream (captured into a CUDA graph
where one is being captured) and nothing synchronises.  Unlike the bridge
calls of `native`, CPU tensors are refused.  Inference only: no gradients.
Wrong shapes, types and devices raise ValueError, a failing call RuntimeError.
Indexes that only the device knows (slots, pages, lengths, positions) are
checked by the kernels, which skip what is out of range and set code 512 in
the device error word (moe_b200_device_error).
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import native

_CODE = {torch.float32: native.DTYPE_F32, torch.bfloat16: native.DTYPE_BF16, torch.float16: native.DTYPE_F16}
_FP8 = (torch.float8_e4m3fn, torch.uint8, torch.int8)
# The current stream's handle without a Stream object around it (2 us of a 10 us call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


class NormedRows(NamedTuple):
    """rmsnorm_fp8's outputs."""

    codes: torch.Tensor  # e4m3 [..., cols]
    scales: torch.Tensor  # fp32 [..., ceil(cols / 128)]
    residual: torch.Tensor  # the stream that was normalised: x + residual in x's type, or x itself
    normed: torch.Tensor | None  # the normed rows in x's type, when asked for


def _call(fn, index: int, *args) -> None:
    """fn(*args, stream) on device `index`, on its current stream."""
    if index == torch.cuda.current_device():
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        native._check(code, fn.__name__)


def _one_device(*tensors: torch.Tensor | None) -> int:
    """The index of the CUDA device that all of them are on."""
    index = tensors[0].get_device()
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors must be on one device")
    return index


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, cols] with contiguous columns: a view where its strides allow one."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _new_codes(flat: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """Codes [rows, cols] whose rows start on 16-byte boundaries, as fp8_block_linear reads them."""
    if cols % 16 == 0:
        return torch.empty_like(flat, dtype=torch.float8_e4m3fn) if flat.is_contiguous() else flat.new_empty((rows, cols), dtype=torch.float8_e4m3fn)
    return flat.new_empty((rows, (cols + 15) // 16 * 16), dtype=torch.float8_e4m3fn)[:, :cols]


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6,
                return_normed: bool = False) -> NormedRows:
    """h = x + residual (in x's type); y = h / sqrt(mean(h^2) + eps) * weight; y as e4m3 codes with one
    fp32 scale per 128 columns, max(amax, 2^-100) / 448.

    x [..., cols] bf16, fp16 or fp32 (rows of a wider tensor need no copy), cols <= 32768; weight [cols] of x's
    type or fp32; residual like x.  The mean is of h as it is returned.  return_normed adds y in x's type, the
    rows that a router reads."""
    shape, dtype = x.shape, x.dtype
    cols = shape[-1] if shape else 0
    code = _CODE.get(dtype)
    if not (code is not None):
        raise ValueError("x must be bf16, fp16 or fp32")
    if not (cols > 0):
        raise ValueError("x must be [..., cols]")
    if not (weight.shape == (cols,)):
        raise ValueError("weight must be [cols]")
    if not (weight.dtype == dtype or weight.dtype == torch.float32):
        raise ValueError("weight must be of x's type or fp32")
    if not (residual is None or (residual.shape == shape and residual.dtype == dtype)):
        raise ValueError("residual must be like x")
    if not (cols <= 32768):
        raise ValueError("x has more than 32768 columns")
    device = _one_device(x, weight, residual)
    flat, weight = _rows(x), weight.contiguous()
    rows = flat.shape[0]
    codes = _new_codes(flat, rows, cols)
    scales = flat.new_empty((rows, (cols + 127) // 128), dtype=torch.float32)
    normed = flat.new_empty((rows, cols)) if return_normed else None
    stream = res = None
    if residual is not None:
        res, stream = _rows(residual), torch.empty_like(flat) if flat.is_contiguous() else flat.new_empty((rows, cols))
    if rows:
        _call(native.load_library().moe_rmsnorm_fp8, device, flat.data_ptr(), flat.stride(0), code, None if res is None else res.data_ptr(),
              0 if res is None else res.stride(0), weight.data_ptr(), code if weight.dtype == dtype else native.DTYPE_F32,
              rows, cols, eps, codes.data_ptr(), codes.stride(0) if rows > 1 else cols, scales.data_ptr(),
              None if stream is None else stream.data_ptr(), None if normed is None else normed.data_ptr())
    if len(shape) != 2:
        codes, scales = codes.view(shape), scales.view(*shape[:-1], scales.shape[1])
        normed = None if normed is None else normed.view(shape)
        stream = None if stream is None else stream.view(shape)
    return NormedRows(codes, scales, x if stream is None else stream, normed)


def quantize_fp8_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., cols] (bf16, fp16 or fp32) as e4m3 codes [..., cols] with one fp32 scale per 128 columns,
    max(amax, 2^-100) / 448."""
    shape = x.shape
    cols = shape[-1] if shape else 0
    code = _CODE.get(x.dtype)
    if not (code is not None):
        raise ValueError("x must be bf16, fp16 or fp32")
    if not (cols > 0):
        raise ValueError("x must be [..., cols]")
    device = _one_device(x)
    flat = _rows(x)
    rows = flat.shape[0]
    codes = _new_codes(flat, rows, cols)
    scales = flat.new_empty((rows, (cols + 127) // 128), dtype=torch.float32)
    if rows:
        _call(native.load_library().moe_fp8_quantize_rows, device, flat.data_ptr(), flat.stride(0), code, rows, cols, codes.data_ptr(),
              codes.stride(0) if rows > 1 else cols, scales.data_ptr())
    if len(shape) != 2:
        codes, scales = codes.view(shape), scales.view(*shape[:-1], scales.shape[1])
    return codes, scales


def _code_rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, cols] codes whose rows start on 16-byte boundaries (a copy where they do not)."""
    if t.stride(1) == 1 and t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    wide = torch.empty((t.shape[0], (t.shape[1] + 15) // 16 * 16), dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    return wide.copy_(t)


def fp8_block_linear(codes: torch.Tensor, scales: torch.Tensor, fp8_weight: torch.Tensor, scale_inv: torch.Tensor, *,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[t, n] = sum_g scales[t, g] scale_inv[n // 128, g] sum_{k in group g} codes[t, k] fp8_weight[n, k].

    codes [..., in] and scales [..., ceil(in / 128)] as rmsnorm_fp8 and quantize_fp8_rows give them; fp8_weight
    [out, in] e4m3 (or its bytes) and scale_inv [ceil(out / 128), ceil(in / 128)] as the checkpoints hold them.
    Sums in fp32, one rounding to out_dtype (bf16, fp16 or fp32).  NaN codes are NaN (the fp32-activation linears
    of `native` read them as 0).  Rows that do not start on 16-byte boundaries are copied first.  The sums' order goes
    by the sizes, so that a row's last bits may be others beside more or fewer rows (never from run to run)."""
    if not (codes.dtype in _FP8 and fp8_weight.dtype in _FP8):
        raise ValueError("codes and fp8_weight must be e4m3")
    if not (scales.dtype == torch.float32 and scale_inv.dtype == torch.float32):
        raise ValueError("scales must be fp32")
    if not (out_dtype in _CODE):
        raise ValueError("out_dtype must be bf16, fp16 or fp32")
    if not (fp8_weight.ndim == 2):
        raise ValueError("fp8_weight must have shape [out_rows, in_cols]")
    if not (scale_inv.ndim == 2):
        raise ValueError("scale_inv must have shape [scale_rows, scale_cols]")
    outs, cols = fp8_weight.shape
    blocks = (cols + 127) // 128
    if not (outs > 0 and cols > 0):
        raise ValueError("fp8_weight must not be empty")
    if not (codes.ndim >= 1 and codes.shape[-1] == cols):
        raise ValueError("hidden input size does not match FP8 weight columns")
    if not (scale_inv.shape == ((outs + 127) // 128, blocks)):
        raise ValueError("scale_inv shape does not match FP8 128x128 block layout")
    lead = codes.shape[:-1]
    if not (scales.shape == (*lead, blocks)):
        raise ValueError("scales must be [..., ceil(in_cols / 128)]")
    device = _one_device(codes, scales, fp8_weight, scale_inv)
    x, w = codes if codes.ndim == 2 else codes.reshape(-1, cols), _code_rows(fp8_weight)
    rows = x.shape[0]
    x, scales, scale_inv = _code_rows(x), scales.contiguous(), scale_inv.contiguous()
    out = scales.new_empty((rows, outs), dtype=out_dtype)
    if rows:
        _call(native.load_library().moe_fp8_block_linear, device, x.data_ptr(), x.stride(0), scales.data_ptr(), w.data_ptr(), w.stride(0),
              scale_inv.data_ptr(), rows, outs, cols, out.data_ptr(), _CODE[out_dtype])
    return out if len(lead) == 1 else out.reshape(*lead, outs)


def _cache_layout(cache: torch.Tensor):
    shape, strides, dtype = cache.shape, cache.stride(), cache.dtype
    if len(shape) != 3 or strides[2] != 1 or 0 in shape:
        raise ValueError("cache must be [pages, page_size, latent + rope]")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError("cache must be bf16 or fp16")
    return *shape, dtype, strides


def paged_mla_append(kv_rows: torch.Tensor, kv_norm_weight: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
                     positions: torch.Tensor, rope_cos: torch.Tensor, rope_sin: torch.Tensor, *, eps: float = 1e-6,
                     q_pe: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores tokens' rows [RMSNorm(kv[:latent]) * kv_norm_weight, rot(kv[latent:], position)] in `cache`, in place,
    and returns the queries' rope parts rotated by the same positions (None without q_pe).

    kv_rows [tokens, latent + rope] (the kv_a projection's rows; a slice of wider ones needs no copy) and
    kv_norm_weight [latent] of the cache's type or fp32; cache [pages, page_size, latent + rope] bf16 or fp16;
    slots int64 [tokens] = page * page_size + offset, distinct, negative for rows to leave out; positions int64
    [tokens] into rope_cos / rope_sin fp32 [max_positions, rope / 2], pairs (2p, 2p + 1); q_pe [tokens, heads,
    rope] of the cache's type (a slice of the q_b projection's output needs no copy).  A position outside the
    tables gives zero queries and stores no row."""
    pages, page_size, width, dtype, strides = _cache_layout(cache)
    code, kv_shape, table = _CODE[dtype], kv_rows.shape, rope_cos.shape
    if kv_norm_weight.ndim != 1 or len(table) != 2 or table != rope_sin.shape:
        raise ValueError("kv_norm_weight must be [latent], rope_cos and rope_sin [max_positions, rope / 2]")
    latent, rope = kv_norm_weight.shape[0], 2 * table[1]
    if len(kv_shape) != 2 or kv_shape[1] != width or latent + rope != width:
        raise ValueError("kv_rows, cache and norm weight sizes do not match")
    if latent == 0 or rope == 0 or table[0] == 0:
        raise ValueError("latent, rope and the tables must not be empty")
    tokens = kv_shape[0]
    if slots.shape != (tokens,) or positions.shape != (tokens,):
        raise ValueError("slots and positions must be [tokens]")
    if slots.dtype != torch.int64 or positions.dtype != torch.int64:
        raise ValueError("slots and positions must be int64")
    kv_code, norm_code = _CODE.get(kv_rows.dtype), _CODE.get(kv_norm_weight.dtype)
    if kv_code != code and kv_code != native.DTYPE_F32:
        raise ValueError("kv_rows must be of the cache's type or fp32")
    if norm_code != code and norm_code != native.DTYPE_F32:
        raise ValueError("kv_norm_weight must be of the cache's type or fp32")
    if rope_cos.dtype != torch.float32 or rope_sin.dtype != torch.float32:
        raise ValueError("rope tables must be fp32")
    heads, q_ptr, q_strides, q_out = 0, None, (0, 0), None
    if q_pe is not None:
        q_shape = q_pe.shape
        if len(q_shape) != 3 or q_shape[0] != tokens or q_shape[1] == 0 or q_shape[2] != rope:
            raise ValueError("q_pe must be [tokens, heads, rope]")
        if q_pe.dtype != dtype:
            raise ValueError("q_pe must be of the cache's type")
        heads = q_shape[1]
    device = _one_device(cache, kv_rows, kv_norm_weight, slots, positions, rope_cos, rope_sin, q_pe)
    if q_pe is not None:
        q_strides = q_pe.stride()
        if q_strides[2] != 1:
            q_pe = q_pe.contiguous()
            q_strides = q_pe.stride()
        q_ptr, q_out = q_pe.data_ptr(), cache.new_empty((tokens, heads, rope))
    if tokens:
        kv, norm_w, slots, positions = _rows(kv_rows), kv_norm_weight.contiguous(), slots.contiguous(), positions.contiguous()
        cos, sin = rope_cos.contiguous(), rope_sin.contiguous()
        _call(native.load_library().moe_paged_mla_append, device, kv.data_ptr(), kv.stride(0), kv_code, norm_w.data_ptr(),
              norm_code, slots.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), table[0], cache.data_ptr(),
              code, pages, page_size, strides[0], strides[1], q_ptr, q_strides[0], q_strides[1], heads,
              None if q_out is None else q_out.data_ptr(), tokens, latent, rope, eps)
    return q_out


@functools.lru_cache(maxsize=256)
def _attention_workspace(*dims: int) -> int:
    return max(int(native.load_library().moe_paged_mla_attention_workspace_bytes(*dims)), 256)


def _query(t: torch.Tensor) -> tuple[torch.Tensor, int, tuple[int, ...]]:
    """Queries whose rows start on 16-byte boundaries and are stored one by one (a copy where they are not), with their
    address and strides."""
    strides, ptr = t.stride(), t.data_ptr()
    if strides[2] != 1 or strides[0] <= 0 or strides[1] <= 0 or strides[0] % 8 or strides[1] % 8 or ptr % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        strides, ptr = t.stride(), t.data_ptr()
    return t, ptr, strides


def paged_mla_attention(q_latent: torch.Tensor, q_pe: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor,
                        lengths: torch.Tensor, *, softmax_scale: float, return_lse: bool = False):
    """Attention of one new token per row over its pages of a latent cache, in the absorbed form:
    score = softmax_scale * (q_latent . latent + q_pe . rope part), out = softmax(score) . latent.

    q_latent [batch, heads, latent] (W_UK^T q_nope), q_pe [batch, heads, rope] (rotated) and cache [pages,
    page_size, latent + rope], all bf16 or all fp16; page_table int32 [batch, max_pages], lengths int32 [batch]
    (the new token included).  Returns [batch, heads, latent] in the queries' type, for W_UV, and with
    return_lse also log(sum exp(score)) fp32 [batch, heads].  A row of length 0 gives zeros (and -inf); entries of
    page_table past a row's last page are not read.  Several tokens of one sequence are rows with the same pages and
    lengths one apart.  latent <= 512 and rope <= 64, multiples of 8; any page size.

    Scores, sums and their parts are fp32; the probabilities are rounded to the cache's type before they multiply the
    latent rows, half a step each.  Where a row's positions are cut into parts goes by all rows' lengths, so that its
    last bits may be others in another batch (never from run to run)."""
    pages, page_size, width, dtype, strides = _cache_layout(cache)
    q_shape, pe_shape, table_shape = q_latent.shape, q_pe.shape, page_table.shape
    if len(q_shape) != 3 or len(pe_shape) != 3:
        raise ValueError("q_latent and q_pe must be [batch, heads, dim]")
    batch, heads, latent = q_shape
    rope = pe_shape[2]
    if pe_shape[0] != batch or pe_shape[1] != heads or heads == 0:
        raise ValueError("batch or head count mismatch")
    if latent == 0 or rope == 0 or latent + rope != width:
        raise ValueError("query and cache sizes do not match")
    if q_latent.dtype != dtype or q_pe.dtype != dtype:
        raise ValueError("queries must be of the cache's type")
    if len(table_shape) != 2 or table_shape[0] != batch or table_shape[1] == 0:
        raise ValueError("page_table must be [batch, max_pages]")
    if lengths.shape != (batch,):
        raise ValueError("lengths must be [batch]")
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError("page_table and lengths must be int32")
    cache_ptr = cache.data_ptr()
    if strides[0] % 8 or strides[1] % 8 or cache_ptr % 16:
        raise ValueError("cache rows must start on 16-byte boundaries")
    device = _one_device(cache, q_latent, q_pe, page_table, lengths)
    out = torch.empty_like(q_latent) if q_latent.is_contiguous() else cache.new_empty(q_shape)
    lse = cache.new_empty((batch, heads), dtype=torch.float32) if return_lse else None
    if batch:
        (ql, ql_ptr, ql_strides), (qp, qp_ptr, qp_strides) = _query(q_latent), _query(q_pe)
        table = page_table if page_table.stride(1) == 1 else page_table.contiguous()
        lengths = lengths.contiguous()
        need = _attention_workspace(batch, heads, latent, rope, table_shape[1], page_size)
        work = cache.new_empty((need,), dtype=torch.uint8)
        _call(native.load_library().moe_paged_mla_attention, device, ql_ptr, ql_strides[0], ql_strides[1], qp_ptr,
              qp_strides[0], qp_strides[1], cache_ptr, _CODE[dtype], pages, page_size, strides[0], strides[1],
              table.data_ptr(), table.stride(0), table_shape[1], lengths.data_ptr(), batch, heads, latent, rope,
              softmax_scale, out.data_ptr(), None if lse is None else lse.data_ptr(), work.data_ptr(), need)
    return (out, lse) if return_lse else out
