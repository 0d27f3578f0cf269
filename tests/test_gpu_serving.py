"""The batched operators of pocketlm_b200.serving on the GPU against their
64-bit forms (tests/serving_oracle.py), at the sizes, strides and masks where
they can go wrong; streams, graphs, indexes out of range, and all of them in a row
as a decode step uses them.  Every tolerance is a count of roundings."""

import ctypes
import math

import pytest
import torch

import serving_oracle as oracle
from pocketlm_b200 import native, serving
from test_serving_host import LINEAR_TILES

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
# an fp32 mean of squares, root, quotient and products: at most 70 additions in a row halved by the root, and eight more steps
NORM_REL = (70 / 2 + 8) * oracle.F32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _error_word():
    return native.load_library().moe_b200_device_error(native._stream())


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    _error_word()
    yield
    assert _error_word() == 0


# ------------------------------------------------------------------ norm, quant

@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("rows,cols,pad,residual", [
    (1, 7168, 0, True), (3, 1, 0, False), (5, 127, 0, True), (130, 129, 7, False), (64, 1536, 576, False), (9, 2048, 8, True),
    (2, 8192, 0, True), (3, 8200, 0, False), (2, 16385, 0, True), (1, 32768, 0, False), (700, 520, 0, True)])
def test_rmsnorm(dtype, rows, cols, pad, residual):
    g = _gen(rows * 31 + cols)
    x = (3 * _rnd(g, rows, cols + pad)).to(dtype)[:, :cols]
    w = (1 + 0.1 * _rnd(g, cols)).to(dtype if cols % 2 else f32)
    res = (2 * _rnd(g, rows, cols)).to(dtype) if residual else None
    got = serving.rmsnorm_fp8(x, w, residual=res, eps=1e-6, return_normed=True)
    h, y = oracle.rmsnorm(x, w, res, 1e-6)
    assert torch.equal(got.residual, h) and got.residual.dtype == dtype
    oracle.check_codes(got.codes, got.scales, y, NORM_REL)
    assert got.normed.dtype == dtype
    off = (got.normed.double() - y).abs()
    assert bool((off <= y.abs() * (oracle.half(dtype) + 2 * NORM_REL) + oracle.least(dtype)).all())


@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("rows,cols,pad", [(1, 128, 0), (1, 1, 0), (7, 130, 3), (64, 16384, 0), (33, 7000, 8), (513, 264, 0)])
def test_quantize(dtype, rows, cols, pad):
    g = _gen(rows + cols)
    x = (_rnd(g, rows, cols + pad) * torch.exp(3 * _rnd(g, rows, 1))).to(dtype)[:, :cols]
    codes, scales = serving.quantize_fp8_rows(x)
    oracle.check_codes(codes, scales, x.double(), 3 * oracle.F32)
    assert codes.stride(0) % 16 == 0


def test_groups_without_values_and_without_numbers():
    x = torch.zeros(4, 384, device="cuda", dtype=bf16)
    x[1, 5], x[2, 200], x[3, 300] = 1e-38, math.inf, math.nan
    codes, scales = serving.quantize_fp8_rows(x)
    c, s = codes.float(), scales
    tiny = torch.tensor(oracle.TINY / 448, device="cuda")
    assert torch.equal(c[0], torch.zeros_like(c[0])) and torch.allclose(s[0], tiny)
    assert not c[1].isnan().any() and s[1].isfinite().all()
    assert s[2, 1].isinf() and c[2, 200].isnan() and int((c[2, 128:256] != 0).sum()) == 1 and not c[2, :128].isnan().any()
    assert s[3, 2].isnan() and c[3, 256:].isnan().all() and not c[3, :256].isnan().any()
    n = serving.rmsnorm_fp8(x, torch.ones(384, device="cuda"), return_normed=True)
    assert not n.codes[:2].float().isnan().any() and n.codes[3].float().isnan().all() and n.scales[3].isnan().all()


def test_norm_shapes_and_views():
    g = _gen(2)
    x, w = _rnd(g, 2, 3, 200).to(bf16), torch.ones(200, device="cuda", dtype=bf16)
    got, flat = serving.rmsnorm_fp8(x, w, return_normed=True), serving.rmsnorm_fp8(x.reshape(6, 200), w, return_normed=True)
    assert got.codes.shape == x.shape and got.scales.shape == (2, 3, 2) and got.residual is x and got.normed.shape == x.shape
    for a, b in zip(got, flat):
        assert torch.equal(a.reshape(6, -1).float(), b.float())
    one = serving.rmsnorm_fp8(x[0, 0], w)
    assert one.codes.shape == (200,) and torch.equal(one.codes.float(), flat.codes[0].float()) and one.normed is None
    t = _rnd(g, 200, 5).to(bf16).t()  # columns strided
    assert torch.equal(serving.rmsnorm_fp8(t, w).codes.float(), serving.rmsnorm_fp8(t.contiguous(), w).codes.float())
    same = x[:1, 0].expand(4, 200)  # rows of stride 0
    assert torch.equal(serving.quantize_fp8_rows(same)[0].float(), serving.quantize_fp8_rows(same.contiguous())[0].float())
    none = serving.rmsnorm_fp8(x[:0], w, residual=x[:0])
    assert none.codes.shape == (0, 3, 200) and none.scales.shape == (0, 3, 2) and none.residual.shape == (0, 3, 200)
    assert serving.quantize_fp8_rows(x[:0])[1].shape == (0, 3, 2)


# ----------------------------------------------------------------------- linear

def _linear_inputs(rows, outs, cols, seed=0):
    g = _gen(rows + outs * 3 + cols * 7 + seed)
    codes, scales = serving.quantize_fp8_rows(_rnd(g, rows, cols))
    w = (100 * _rnd(g, outs, cols)).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = torch.rand((outs + 127) // 128, (cols + 127) // 128, generator=g, device="cuda") * 1e-3 + 1e-4
    return codes, scales, w, ws


def _check_linear(out, codes, scales, w, ws):
    want, size = oracle.linear(codes, scales, w, ws)
    # fp32 sums: at most 128 products in a group's row and one scaled addition per group, each at worst a step;
    # the scales' product rounded too
    steps = 128 + scales.shape[-1] + 4
    tol = size * steps * 2 * oracle.F32 + want.abs() * oracle.half(out.dtype) + oracle.least(out.dtype)
    assert bool(((out.double() - want).abs() <= tol).all())
    # and on the whole nearly as exact as the output's type: rounding errors add up like sqrt(steps) at random
    rel = float((out.double() - want).norm() / want.norm())
    assert rel <= oracle.half(out.dtype) + math.sqrt(steps) * 4 * oracle.F32


@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("rows,outs,cols", [
    (1, 1, 16), (1, 2112, 7168), (3, 576, 1536), (16, 128, 128), (17, 130, 257), (33, 257, 4096), (64, 1000, 1536), (65, 300, 520),
    (127, 384, 640), (128, 256, 2048), (129, 513, 1111), (200, 128, 8192), (257, 1100, 384), (600, 640, 1024)])
def test_linear(dtype, rows, outs, cols):
    args = _linear_inputs(rows, outs, cols)
    _check_linear(serving.fp8_block_linear(*args, out_dtype=dtype), *args)


def test_linear_large():
    args = _linear_inputs(1500, 7168, 2048)
    out = serving.fp8_block_linear(*args)
    _check_linear(out, *args)
    assert torch.equal(out, serving.fp8_block_linear(*args))  # sums do not depend on who comes first


@pytest.mark.parametrize("rows,outs,cols", [(100, 1003, 4096), (64, 5001, 640), (9, 387, 2064), (300, 1030, 1000)])
def test_linear_few_rows_of_odd_outputs(rows, outs, cols):
    """Outputs that are not stored four at a time, with a cluster's sums and without."""
    args = _linear_inputs(rows, outs, cols)
    for dtype in (bf16, f32):
        out = serving.fp8_block_linear(*args, out_dtype=dtype)
        _check_linear(out, *args)
        assert torch.equal(out, serving.fp8_block_linear(*args, out_dtype=dtype))


def test_linear_strides_and_shapes():
    codes, scales, w, ws = _linear_inputs(24, 200, 300)
    want = serving.fp8_block_linear(codes, scales, w, ws)
    bytes_ = serving.fp8_block_linear(codes.view(torch.uint8), scales, w.view(torch.uint8), ws)
    assert torch.equal(bytes_, want)
    packed = codes.contiguous()  # rows of 300 bytes: copied to 16-byte boundaries first
    assert packed.stride(0) == 300 and torch.equal(serving.fp8_block_linear(packed, scales, w, ws), want)
    wide = torch.empty(200, 320, dtype=w.dtype, device="cuda")[:, :300]
    wide.copy_(w)
    assert torch.equal(serving.fp8_block_linear(codes, scales.t().contiguous().t(), wide, ws), want)
    cube = serving.fp8_block_linear(packed.view(2, 12, 300), scales.view(2, 12, 3), w, ws)
    assert cube.shape == (2, 12, 200) and torch.equal(cube.view(24, 200), want)
    assert serving.fp8_block_linear(codes[0], scales[0], w, ws).shape == (200,)
    assert serving.fp8_block_linear(codes[:0], scales[:0], w, ws).shape == (0, 200)


def test_linear_nan_codes_stay_in_their_rows():
    codes, scales, w, ws = _linear_inputs(20, 256, 256)
    codes, w = codes.clone(), w.clone()
    codes.view(torch.uint8)[3, 7] = 0x7F
    w.view(torch.uint8)[100, 200] = 0xFF
    out = serving.fp8_block_linear(codes, scales, w, ws, out_dtype=f32).isnan()
    assert bool(out[3].all()) and bool(out[:, 100].all())
    out[3], out[:, 100] = False, False
    assert not out.any()


def _tile(rows, outs, cols):
    return native.load_library().moe_fp8_block_linear_tile(rows, outs, cols)


def _of_148_sms():
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("shapes chosen for the tiles that 148 SMs take")


# outputs that are no multiple of a vector, a tile or a weight block, columns that end inside a group, a pair whose second CTA
# has no tokens (rows % 256 up to 128), several tiles per CTA; and whole ones
@pytest.mark.parametrize("dtype", [bf16, f16, f32])
@pytest.mark.parametrize("tile,rows,outs,cols", LINEAR_TILES)
def test_linear_every_tile(dtype, tile, rows, outs, cols):
    _of_148_sms()
    assert _tile(rows, outs, cols) == tile
    args = _linear_inputs(rows, outs, cols)
    out = serving.fp8_block_linear(*args, out_dtype=dtype)
    _check_linear(out, *args)
    assert torch.equal(out, serving.fp8_block_linear(*args, out_dtype=dtype))


@pytest.mark.parametrize("rows,outs,cols", [(513, 5377, 333), (257, 7109, 515), (129, 4745, 333), (514, 6163, 333)])
def test_linear_nan_codes_stay_in_their_rows_of_every_tile(rows, outs, cols):
    codes, scales, w, ws = _linear_inputs(rows, outs, cols)
    codes, w = codes.clone(), w.clone()
    codes.view(torch.uint8)[rows - 1, cols - 1] = 0x7F
    w.view(torch.uint8)[outs - 2, 5] = 0xFF
    out = serving.fp8_block_linear(codes, scales, w, ws, out_dtype=f32).isnan()
    assert bool(out[rows - 1].all()) and bool(out[:, outs - 2].all())
    out[rows - 1], out[:, outs - 2] = False, False
    assert not out.any()


@pytest.mark.parametrize("rows,outs,cols", [(1, 3, 2225152), (17, 3, 1030144), (33, 5, 531456), (65, 130, 68608)])
def test_linear_more_groups_than_scales_fit(rows, outs, cols):
    """The longest rows whose scales stay in shared memory, and one column more."""
    _of_148_sms()
    assert _tile(rows, outs, cols) % 1000 == 128 and _tile(rows, outs, cols + 1) == 256192
    for k in (cols, cols + 1):
        args = _linear_inputs(rows, outs, k)
        _check_linear(serving.fp8_block_linear(*args, out_dtype=f32), *args)


# ----------------------------------------------------------------------- append

def _append_case(tokens, heads, latent, rope, page, cache_dtype, kv_dtype, pad=0, seed=0):
    g = _gen(tokens * 7 + heads + latent + seed)
    pages = (2 * tokens) // page + 3
    cache = _rnd(g, pages, page, latent + rope + pad).to(cache_dtype)[..., :latent + rope]
    kv = (2 * _rnd(g, tokens, latent + rope + 40)).to(kv_dtype)[:, 40:]
    w = (1 + 0.1 * _rnd(g, latent)).to(f32 if heads % 2 else cache_dtype)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2::5] = -1
    pos = torch.randint(0, 999, (tokens,), generator=g, device="cuda")
    angle = torch.arange(999, device="cuda", dtype=torch.float64)[:, None] * torch.rand(rope // 2, generator=g, device="cuda").double()
    q = _rnd(g, tokens, heads, rope + 24).to(cache_dtype)[..., 24:]
    return kv, w, cache, slots, pos, angle.cos().float(), angle.sin().float(), q


def _check_append(before, cache, q_out, kv, w, slots, pos, cos, sin, q):
    latent, page = w.shape[0], cache.shape[1]
    half, least = oracle.half(cache.dtype), oracle.least(cache.dtype)
    _, y = oracle.rmsnorm(kv[:, :latent].float(), w, None, 1e-6)
    c, s = cos.double()[pos], sin.double()[pos]
    r, size = oracle.rotate(kv[:, latent:].double(), c, s)
    want, live = before.double().clone(), slots >= 0
    tol = torch.zeros_like(want)
    where = (slots[live] // page, slots[live] % page)
    want[where] = torch.cat((y, r), 1)[live]
    # the norm's fp32 steps, or two products and a sum; then half a step of the cache's type
    tol[where] = torch.cat((y.abs() * (half + 2 * NORM_REL), size * 3 * oracle.F32 + r.abs() * half), 1)[live] + least
    assert bool(((cache.double() - want).abs() <= tol).all())
    turned, size = oracle.rotate(q.double(), c[:, None], s[:, None])
    assert bool(((q_out.double() - turned).abs() <= size * 3 * oracle.F32 + turned.abs() * half + least).all())


@pytest.mark.parametrize("cache_dtype,kv_dtype", [(bf16, bf16), (f16, f16), (bf16, f32)])
@pytest.mark.parametrize("tokens,heads,latent,rope,page,pad", [
    (1, 128, 512, 64, 64, 0), (37, 16, 512, 64, 16, 64), (5, 3, 40, 6, 1, 0), (130, 7, 129, 10, 48, 3), (300, 128, 1024, 64, 7, 0),
    (2, 1, 8, 2, 5, 0)])
def test_append(cache_dtype, kv_dtype, tokens, heads, latent, rope, page, pad):
    kv, w, cache, slots, pos, cos, sin, q = _append_case(tokens, heads, latent, rope, page, cache_dtype, kv_dtype, pad)
    before = cache.clone()
    q_out = serving.paged_mla_append(kv, w, cache, slots, pos, cos, sin, eps=1e-6, q_pe=q)
    assert q_out.is_contiguous() and q_out.dtype == cache_dtype
    _check_append(before, cache, q_out, kv, w, slots, pos, cos, sin, q)
    again = before.clone()
    assert serving.paged_mla_append(kv, w, again, slots, pos, cos, sin, eps=1e-6) is None
    assert torch.equal(again, cache)  # with and without queries


def test_append_out_of_range_is_skipped():
    kv, w, cache, slots, pos, cos, sin, q = _append_case(6, 4, 64, 16, 8, bf16, bf16)
    slots = torch.tensor([0, cache.shape[0] * 8, 3, -5, 9, 10], device="cuda")
    pos = torch.tensor([5, 6, 999, -1, -2, 998], device="cuda")
    before = cache.clone()
    q_out = serving.paged_mla_append(kv, w, cache, slots, pos, cos, sin, q_pe=q)
    assert _error_word() == 512
    flat, was = cache.reshape(-1, 80), before.reshape(-1, 80)
    changed = (flat != was).any(1).nonzero().flatten().tolist()
    assert changed == [0, 10]
    assert not q_out[2:5].any() and bool(q_out[[0, 1, 5]].any(2).all())
    # rows to leave out may hold any position: no error
    serving.paged_mla_append(kv, w, cache, torch.full_like(slots, -1), pos, cos, sin)
    assert _error_word() == 0


@pytest.mark.parametrize("tokens,heads,latent,rope", [(1000, 130, 512, 64), (1500, 5, 72, 16), (2000, 33, 40, 10), (900, 1, 16, 280)])
def test_append_many_tokens(tokens, heads, latent, rope):
    """More tokens than CTAs, whose next tokens are read ahead; more heads than a CTA turns at once."""
    kv, w, cache, slots, pos, cos, sin, q = _append_case(tokens, heads, latent, rope, 16, bf16, bf16)
    before = cache.clone()
    q_out = serving.paged_mla_append(kv, w, cache, slots, pos, cos, sin, eps=1e-6, q_pe=q)
    _check_append(before, cache, q_out, kv, w, slots, pos, cos, sin, q)
    lost = pos.clone()
    lost[slots < 0] = 1 << 40  # rows to leave out, without a place in the sequence: zeros, and no error
    q_lost = serving.paged_mla_append(kv, w, cache, slots, lost, cos, sin, eps=1e-6, q_pe=q)
    assert not q_lost[slots < 0].any() and torch.equal(q_lost[slots >= 0], q_out[slots >= 0])


def test_append_no_tokens():
    kv, w, cache, slots, pos, cos, sin, q = _append_case(4, 2, 64, 16, 8, f16, f16)
    before = cache.clone()
    out = serving.paged_mla_append(kv[:0], w, cache, slots[:0], pos[:0], cos, sin, q_pe=q[:0])
    assert out.shape == (0, 2, 16) and torch.equal(before, cache)


# -------------------------------------------------------------------- attention

def _attn_case(lengths, heads, latent, rope, page, dtype, seed=0, spread=1.5, pad=0, slack=0):
    g = _gen(sum(lengths) + heads * 3 + latent + seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 2
    cache = _rnd(g, pages, page, latent + rope + pad).to(dtype)[..., :latent + rope]
    order = torch.randperm(pages, generator=g, device="cuda").int().cpu()
    table = torch.full((len(lengths), max(1, max(need, default=1)) + slack), -7, dtype=torch.int32)  # never read past the last page
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
        if lengths[i] % page:  # the unused end of the last page may hold anything
            cache[int(table[i, n - 1]), lengths[i] % page:] = math.nan
    q = (_rnd(g, len(lengths), heads, latent + rope) * spread).to(dtype)
    return q[..., :latent], q[..., latent:], cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), (latent + rope) ** -0.5


def _check_attn(out, lse, case):
    ql, qp, cache, table, lengths, scale = case
    want, want_lse, tol, lse_tol = oracle.attention(ql, qp, cache.nan_to_num(), table, lengths, scale)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert bool(((out - want).abs() <= tol).all())
    empty = torch.isinf(want_lse)
    assert torch.equal(lse == -math.inf, empty)
    assert bool(((lse - want_lse).abs()[~empty] <= lse_tol[~empty]).all())


@pytest.mark.parametrize("dtype", [bf16, f16])
@pytest.mark.parametrize("lengths,heads,page", [
    ([1], 128, 64), ([64], 128, 64), ([65], 16, 64), ([4096], 128, 64), ([1000, 0, 1, 17, 63], 128, 16), ([300, 7, 128, 129], 16, 48),
    ([5, 77, 200], 1, 1), ([513, 511, 512], 40, 128), ([2000, 33], 129, 7), ([0, 0], 8, 64), ([700], 64, 1024), ([190, 64, 3] * 30, 32, 32)])
def test_attention(dtype, lengths, heads, page):
    case = _attn_case(lengths, heads, 512, 64, page, dtype)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    assert out.dtype == dtype and out.shape == (len(lengths), heads, 512)
    _check_attn(out, lse, case)


@pytest.mark.parametrize("latent,rope", [(8, 8), (64, 16), (128, 32), (200, 40), (256, 64), (448, 8), (504, 56)])
def test_attention_widths(latent, rope):
    case = _attn_case([130, 0, 9, 400], 20, latent, rope, 24, bf16, pad=8)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    _check_attn(out, lse, case)


@pytest.mark.parametrize("latent", [256, 320, 384, 448, 512])
@pytest.mark.parametrize("page", [2, 8, 16, 40, 64, 192])
def test_attention_page_sizes(latent, page):
    """Every way in which rows are copied: single rows, blocks of 8, runs of 64, whole and odd numbers of column chunks."""
    case = _attn_case([300, 129, 0, 64], 70, latent, 64, page, bf16)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    _check_attn(out, lse, case)


@pytest.mark.parametrize("lengths,heads,latent", [([190, 64, 3, 0] * 20, 37, 512), ([700, 129] * 8, 130, 512), ([1, 400, 260] * 15, 41, 72)])
def test_attention_many_rows_of_odd_heads(lengths, heads, latent):
    """Parts joined four heads at a time, of which the last do not exist."""
    case = _attn_case(lengths, heads, latent, 64, 32, f16)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    _check_attn(out, lse, case)
    assert torch.equal(out, serving.paged_mla_attention(*case[:5], softmax_scale=case[5]))


@pytest.mark.parametrize("batch,heads,page", [(257, 16, 16), (300, 129, 64), (600, 5, 7), (1030, 12, 32)])
def test_attention_more_rows_than_threads(batch, heads, page):
    """A thread adds up the tiles of several rows and finds its range's first one among them: long rows and long stretches of
    rows without positions, at both ends and in between."""
    lengths = [(37 * i) % 90 + 1 for i in range(batch)]
    lengths[:9] = [0] * 9
    lengths[60:140] = [0] * 80
    lengths[140], lengths[batch - 2], lengths[batch - 1] = 2500, 1300, 0
    case = _attn_case(lengths, heads, 64, 16, page, bf16)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    _check_attn(out, lse, case)
    assert torch.equal(out, serving.paged_mla_attention(*case[:5], softmax_scale=case[5]))


def test_attention_most_rows():
    """As many rows as a call takes.  A row of one tile is never cut, so that it does not depend on the rows beside it."""
    batch, heads, latent, rope, page = 65535, 3, 64, 16, 16
    g = _gen(9)
    cache = _rnd(g, 1000, page, latent + rope).to(bf16)
    table = torch.randint(0, 1000, (batch, 8), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(0, 129, (batch,), generator=g, device="cuda", dtype=torch.int32)
    lengths[1000:3000] = 0
    q = _rnd(g, batch, heads, latent + rope).to(bf16)
    ql, qp = q[..., :latent].contiguous(), q[..., latent:].contiguous()
    out, lse = serving.paged_mla_attention(ql, qp, cache, table, lengths, softmax_scale=0.1, return_lse=True)
    for at in range(0, batch, 1000):
        rows = slice(at, at + 200)
        few, few_lse = serving.paged_mla_attention(ql[rows], qp[rows], cache, table[rows], lengths[rows], softmax_scale=0.1, return_lse=True)
        assert torch.equal(out[rows], few) and torch.equal(lse[rows], few_lse)
    _check_attn(out[-100:], lse[-100:], (ql[-100:], qp[-100:], cache, table[-100:], lengths[-100:], 0.1))


@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_attention_flat_and_peaked(spread):
    """Equal scores, and scores of which one takes all (its maximum moving along the cache)."""
    case = _attn_case([900, 31], 128, 512, 64, 64, bf16, spread=spread)
    if spread:  # rising scores: the running maximum changes in every tile
        case[2].copy_((case[2].float() * torch.linspace(0.1, 1, case[2].shape[0], device="cuda")[:, None, None]).to(bf16))
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=case[5], return_lse=True)
    _check_attn(out, lse, case)


def test_attention_views_and_zero_scale():
    """Queries as slices of wider rows (copied only where they are not on 16-byte boundaries), a table with room, scale 0."""
    ql, qp, cache, table, lengths, scale = _attn_case([100, 250], 24, 512, 64, 64, bf16, slack=5)
    want = serving.paged_mla_attention(ql, qp, cache, table, lengths, softmax_scale=scale)
    wide = torch.zeros(2, 24, 192, device="cuda", dtype=bf16)
    wide[..., 128:] = qp
    turned = ql.permute(1, 0, 2).contiguous().permute(1, 0, 2)  # [heads, batch, latent] in memory, as a product per head leaves it
    assert torch.equal(serving.paged_mla_attention(turned, wide[..., 128:], cache, table, lengths, softmax_scale=scale), want)
    odd = torch.zeros(2, 24, 513, device="cuda", dtype=bf16)
    odd[..., 1:] = ql
    assert torch.equal(serving.paged_mla_attention(odd[..., 1:], qp, cache, table[:, :4], lengths, softmax_scale=scale), want)
    case = (ql, qp, cache, table, lengths, 0.0)
    _check_attn(*serving.paged_mla_attention(*case[:5], softmax_scale=0.0, return_lse=True), case)


def test_attention_verify_batch_shares_pages():
    """Three new tokens of one sequence: one table row, lengths one apart."""
    ql, qp, cache, table, lengths, scale = _attn_case([515], 128, 512, 64, 64, bf16)
    cache.nan_to_num_(0.5)
    case = (ql.expand(3, -1, -1).contiguous(), qp.expand(3, -1, -1), cache, table.expand(3, -1), lengths.expand(3) - torch.arange(3, device="cuda").int(), scale)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=scale, return_lse=True)
    _check_attn(out, lse, case)


def test_attention_bad_pages_and_lengths():
    """A page outside the cache is left out, a length past the table cut, a negative one is none; each sets code 512 (but the last)."""
    ql, qp, cache, table, lengths, scale = _attn_case([200, 200, 200], 16, 512, 64, 64, bf16)
    cache.nan_to_num_(0.25)
    table[0, 1], table[1, 2] = cache.shape[0], -1
    case = (ql, qp, cache, table, lengths, scale)
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=scale, return_lse=True)
    assert _error_word() == 512
    _check_attn(out, lse, case)
    table[0, 1], table[1, 2] = 0, 0
    lengths[0] = 257
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=scale, return_lse=True)
    assert _error_word() == 512
    _check_attn(out, lse, case)
    lengths[0] = -4
    out, lse = serving.paged_mla_attention(*case[:5], softmax_scale=scale, return_lse=True)
    _check_attn(out, lse, case)
    assert serving.paged_mla_attention(ql[:0], qp[:0], cache, table[:0], lengths[:0], softmax_scale=scale).shape == (0, 16, 512)


def test_attention_infinite_and_nan_values_stay_in_their_rows():
    ql, qp, cache, table, lengths, scale = _attn_case([150, 150, 150], 128, 512, 64, 64, bf16)
    cache.nan_to_num_(0.0)
    cache[int(table[1, 1]), 3, 100] = math.nan
    ql = ql.clone()
    ql[2, 5, 7] = math.inf
    out, lse = serving.paged_mla_attention(ql, qp, cache, table, lengths, softmax_scale=scale, return_lse=True)
    # not bit by bit what row 0 gives alone: where its positions are cut, and so which maximum its rounded
    # probabilities are relative to, goes by the whole batch; what the roundings may cost holds either way
    _check_attn(out[:1], lse[:1], (ql[:1], qp[:1], cache, table[:1], lengths[:1], scale))
    assert bool(out[1, :, 100].isnan().all())
    rest = torch.arange(128, device="cuda") != 5
    assert not out[2, rest].isnan().any() and bool(out[2, 5].isnan().any())


def test_attention_far_pages_of_a_long_cache():
    """Element offsets past 2^32: pages at both ends of an 8.6 GB cache (never read in between)."""
    page, width, pages = 64, 576, 120000
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    cache = torch.empty(pages, page, width, dtype=bf16, device="cuda")
    at = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    g = _gen(5)
    cache[at[0].long()] = _rnd(g, 3, page, width).to(bf16)
    q = _rnd(g, 1, 128, width).to(bf16)
    n = torch.tensor([170], dtype=torch.int32, device="cuda")
    got = serving.paged_mla_attention(q[..., :512], q[..., 512:], cache, at, n, softmax_scale=0.05)
    small = cache[at[0].long()].clone()
    want = serving.paged_mla_attention(q[..., :512], q[..., 512:], small, torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), n, softmax_scale=0.05)
    assert torch.equal(got, want)


# ---------------------------------------------------------- streams and graphs

class _Step:
    """One decode step's attention half for a batch: weights, caches and the calls in order."""

    def __init__(self, batch, heads=16, hidden=1024, q_rank=384, latent=512, rope=64, nope=128, seed=3):
        g = _gen(seed)
        self.heads, self.latent, self.rope, self.nope, self.q_rank = heads, latent, rope, nope, q_rank
        self.w_in, self.w_q, self.w_kv = (1 + 0.1 * _rnd(g, n) for n in (hidden, q_rank, latent))

        def fp8(outs, cols):
            w = _rnd(g, outs, cols) * cols ** -0.5
            s = torch.full(((outs + 127) // 128, (cols + 127) // 128), float(w.abs().max()) / 448, device="cuda")
            return (w / s[0, 0]).to(torch.float8_e4m3fn), s

        self.down, self.up, self.o = fp8(q_rank + latent + rope, hidden), fp8(heads * (nope + rope), q_rank), fp8(hidden, heads * 128)
        self.w_uk = (_rnd(g, heads, nope, latent) * nope ** -0.5).to(bf16)
        self.w_uv = (_rnd(g, heads, latent, 128) * latent ** -0.5).to(bf16)
        self.x, self.res = _rnd(g, batch, hidden).to(bf16), _rnd(g, batch, hidden).to(bf16)
        self.lengths = torch.tensor([1 + (97 * i) % 300 for i in range(batch)], dtype=torch.int32, device="cuda")
        self.page, per = 32, 10
        self.cache = _rnd(g, batch * per, self.page, latent + rope).to(bf16)
        self.table = torch.randperm(batch * per, generator=g, device="cuda").int().view(batch, per)
        self.pos = (self.lengths - 1).long()
        self.slots = self.table.gather(1, (self.pos // self.page)[:, None])[:, 0].long() * self.page + self.pos % self.page
        angle = torch.arange(512, device="cuda", dtype=torch.float64)[:, None] * 10000 ** (-torch.arange(0, rope, 2, device="cuda").double() / rope)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.scale = (nope + rope) ** -0.5

    def run(self):
        n = serving.rmsnorm_fp8(self.x, self.w_in, residual=self.res)
        a = serving.fp8_block_linear(n.codes, n.scales, *self.down)
        qn = serving.rmsnorm_fp8(a[:, :self.q_rank], self.w_q)
        q = serving.fp8_block_linear(qn.codes, qn.scales, *self.up).view(-1, self.heads, self.nope + self.rope)
        q_pe = serving.paged_mla_append(a[:, self.q_rank:], self.w_kv, self.cache, self.slots, self.pos, self.cos, self.sin, q_pe=q[..., self.nope:])
        q_lat = torch.bmm(q[..., :self.nope].transpose(0, 1), self.w_uk).transpose(0, 1)
        out = serving.paged_mla_attention(q_lat, q_pe, self.cache, self.table, self.lengths, softmax_scale=self.scale)
        o = torch.bmm(out.transpose(0, 1), self.w_uv).transpose(0, 1).reshape(-1, self.heads * 128)
        return serving.fp8_block_linear(*serving.quantize_fp8_rows(o), *self.o), n.residual

    def plain(self):
        """The same in 64 bits, with the roundings that the calls store (codes and 16-bit results)."""
        def q8(y):
            s = oracle.group_scales(y).float()
            w = s.repeat_interleave(128, 1)[:, :y.shape[1]].double()
            return (y / w).float().to(torch.float8_e4m3fn), s

        def lin(rows, weight):
            return oracle.linear(*rows, *weight)[0].to(bf16)

        h, y = oracle.rmsnorm(self.x, self.w_in, self.res, 1e-6)
        a = lin(q8(y), self.down)
        q = lin(q8(oracle.rmsnorm(a[:, :self.q_rank], self.w_q, None, 1e-6)[1]), self.up).view(-1, self.heads, self.nope + self.rope)
        c, s = self.cos.double()[self.pos], self.sin.double()[self.pos]
        row = torch.cat((oracle.rmsnorm(a[:, self.q_rank:self.q_rank + self.latent], self.w_kv, None, 1e-6)[1],
                         oracle.rotate(a[:, self.q_rank + self.latent:].double(), c, s)[0]), 1).to(bf16)
        cache = self.cache.clone()
        cache[self.slots // self.page, self.slots % self.page] = row
        q_pe = oracle.rotate(q[..., self.nope:].double(), c[:, None], s[:, None])[0].to(bf16)
        q_lat = torch.einsum("bhn,hnr->bhr", q[..., :self.nope].double(), self.w_uk.double()).to(bf16)
        out = oracle.attention(q_lat, q_pe, cache, self.table, self.lengths, self.scale)[0].cuda().to(bf16)
        o = torch.einsum("bhr,hrv->bhv", out.double(), self.w_uv.double()).to(bf16).flatten(1)
        return lin(q8(o.double()), self.o), h, cache


@pytest.mark.parametrize("batch", [1, 5, 70])
def test_a_decode_step(batch):
    step = _Step(batch)
    out, res = step.run()
    want, want_res, cache = step.plain()
    assert torch.equal(res, want_res)
    # both sides round the same six results to 16 bits and three times to e4m3; where a value lies near a border they
    # may round apart, by a step: of the 8-bit codes a share of about 2^-7 / 2^-3 (the 16-bit neighbours over the
    # codes' distance), a step being 2^-3: sqrt(2^-4) 2^-3 / sqrt(3) = 2e-2 per linear at the most, three of them
    rel = float((out.double() - want.double()).norm() / want.double().norm())
    assert rel <= 3 ** 0.5 * 2e-2
    far = float((step.cache.double() - cache.double()).norm() / cache.double().norm())
    assert far <= 2e-2


@pytest.mark.parametrize("batch", [1, 5, 70])
def test_what_a_decode_step_appends(batch):
    """Each sequence's new row, by itself; every other row of the cache bit for bit as it was."""
    step = _Step(batch)
    before = step.cache.clone()
    step.run()
    want = step.plain()[2]
    where = (step.slots // step.page, step.slots % step.page)
    new, row = step.cache[where].double(), want[where].double()
    # one linear of 8-bit codes lies before the row (2e-2 as above), and two roundings to 16 bits that may go apart by a step each
    rel = (new - row).norm(dim=1) / row.norm(dim=1)
    assert float(rel.max()) <= 2e-2 + 2 * 2 * oracle.half(bf16)
    rest = step.cache.clone()
    rest[where] = before[where]
    assert torch.equal(rest, before)


def test_a_decode_step_in_a_graph_and_on_another_stream():
    step = _Step(6)
    before = step.cache.clone()
    want, _ = step.run()
    after = step.cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step.cache.copy_(before)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = step.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(step.cache, after)
    graphs = []
    for _ in range(2):  # two graphs of the same step, replayed in turn: neither uses what the other keeps
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, _ = step.run()
        graphs.append((g, out))
    x = step.x.clone()
    for _ in range(2):
        for g, out in graphs:
            step.x.copy_(x)
            g.replay()
            assert torch.equal(out, want)
            step.x.copy_(2 * x[torch.randperm(6, device="cuda")])
            g.replay()
    step.x.copy_(x)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(step.cache, after)


def test_two_calls_at_once_on_two_streams():
    cases = [_attn_case([3000, 500], 128, 512, 64, 64, bf16, seed=s) for s in (1, 2)]
    linears = [_linear_inputs(40, 2112, 7168, seed=s) for s in (1, 2)]
    want = [(serving.paged_mla_attention(*c[:5], softmax_scale=c[5]), serving.fp8_block_linear(*a)) for c, a in zip(cases, linears)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                c = cases[i]
                got[i].append((serving.paged_mla_attention(*c[:5], softmax_scale=c[5]), serving.fp8_block_linear(*linears[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_c_entry_allocates_its_own_workspace():
    """The C attention call without a workspace gives what the call with one gives."""
    ql, qp, cache, table, lengths, scale = _attn_case([900, 40], 128, 512, 64, 64, bf16)
    ql, qp = ql.contiguous(), qp.contiguous()
    want = serving.paged_mla_attention(ql, qp, cache, table, lengths, softmax_scale=scale)
    out = torch.empty_like(want)
    p = native._ptr
    code = native.load_library().moe_paged_mla_attention(
        p(ql), ql.stride(0), ql.stride(1), p(qp), qp.stride(0), qp.stride(1), p(cache), 1, cache.shape[0], 64, cache.stride(0),
        cache.stride(1), p(table), table.stride(0), table.shape[1], p(lengths), 2, 128, 512, 64, scale, p(out), None,
        ctypes.c_void_p(0), 0, native._stream())
    assert code == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)
