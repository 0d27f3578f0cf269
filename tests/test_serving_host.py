"""The refusals of pocketlm_b200.serving and of its C entry points, on the host:
every call below returns from its argument checks."""

import ctypes

import pytest
import torch

from pocketlm_b200 import native, serving

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced
bf16, f16, f32, i32, i64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64


def _refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_norm_refusals():
    x, w = torch.zeros(4, 256, dtype=bf16), torch.ones(256, dtype=bf16)
    _refused("CUDA device", serving.rmsnorm_fp8, x, w)
    _refused("x must be bf16", serving.rmsnorm_fp8, x.double(), w)
    _refused("weight must be \\[cols\\]", serving.rmsnorm_fp8, x, w[:128])
    _refused("weight must be of", serving.rmsnorm_fp8, x, w.half())
    _refused("residual must be like", serving.rmsnorm_fp8, x, w, residual=x[:2])
    _refused("residual must be like", serving.rmsnorm_fp8, x, w, residual=x.float())
    _refused("32768", serving.rmsnorm_fp8, torch.zeros(1, 32769, dtype=bf16), torch.ones(32769))
    _refused("cols", serving.rmsnorm_fp8, torch.zeros(4, 0), torch.ones(0))
    _refused("CUDA device", serving.quantize_fp8_rows, x)
    _refused("x must be bf16", serving.quantize_fp8_rows, x.long())


def test_linear_refusals():
    c, s = torch.zeros(3, 300, dtype=torch.uint8), torch.ones(3, 3)
    w, ws = torch.zeros(200, 300, dtype=torch.uint8), torch.ones(2, 3)
    _refused("CUDA device", serving.fp8_block_linear, c, s, w, ws)
    _refused("e4m3", serving.fp8_block_linear, c.float(), s, w, ws)
    _refused("fp32", serving.fp8_block_linear, c, s.half(), w, ws)
    _refused("out_dtype", serving.fp8_block_linear, c, s, w, ws, out_dtype=torch.float64)
    _refused("hidden input size", serving.fp8_block_linear, c[:, :256], s[:, :2], w, ws)
    _refused("block layout", serving.fp8_block_linear, c, s, w, ws[:1])
    _refused("scales must be", serving.fp8_block_linear, c, s[:, :2], w, ws)


def _append_args(tokens=5, latent=64, rope=16, heads=3, dtype=bf16):
    return dict(kv_rows=torch.zeros(tokens, latent + rope, dtype=dtype), kv_norm_weight=torch.ones(latent, dtype=dtype),
                cache=torch.zeros(4, 8, latent + rope, dtype=dtype), slots=torch.arange(tokens),
                positions=torch.arange(tokens), rope_cos=torch.ones(32, rope // 2), rope_sin=torch.zeros(32, rope // 2),
                q_pe=torch.zeros(tokens, heads, rope, dtype=dtype))


@pytest.mark.parametrize("change,match", [
    ({}, "CUDA device"), (dict(cache=torch.zeros(4, 8, 80)), "cache must be bf16"),
    (dict(cache=torch.zeros(4, 80, 8, dtype=bf16).transpose(1, 2)), "cache must be \\["),
    (dict(kv_rows=torch.zeros(5, 72, dtype=bf16)), "sizes do not match"), (dict(kv_rows=torch.zeros(5, 80, dtype=f16)), "kv_rows must be of"),
    (dict(slots=torch.arange(4)), "slots and positions"), (dict(slots=torch.arange(5, dtype=i32)), "int64"),
    (dict(rope_cos=torch.ones(32, 8, dtype=f16)), "must be fp32"), (dict(rope_sin=torch.ones(31, 8)), "rope_cos and rope_sin"),
    (dict(q_pe=torch.zeros(5, 3, 8, dtype=bf16)), "q_pe must be \\["), (dict(q_pe=torch.zeros(5, 3, 16)), "q_pe must be of"),
    (dict(kv_norm_weight=torch.ones(64, dtype=f16)), "kv_norm_weight must be of")])
def test_append_refusals(change, match):
    _refused(match, serving.paged_mla_append, **{**_append_args(), **change})


@pytest.mark.parametrize("name", [k for k, v in _append_args().items()])
def test_append_refuses_other_numbers_of_dimensions(name):
    given = _append_args()[name]
    for bad in (given.new_zeros(()), given[None]):
        with pytest.raises(ValueError) as refusal:
            serving.paged_mla_append(**{**_append_args(), name: bad})
        assert "CUDA device" not in str(refusal.value)  # not for where the tensors are


def _attn_args(batch=2, heads=3, latent=64, rope=16, dtype=bf16):
    return dict(q_latent=torch.zeros(batch, heads, latent, dtype=dtype), q_pe=torch.zeros(batch, heads, rope, dtype=dtype),
                cache=torch.zeros(4, 8, latent + rope, dtype=dtype), page_table=torch.zeros(batch, 2, dtype=i32),
                lengths=torch.ones(batch, dtype=i32), softmax_scale=0.1)


@pytest.mark.parametrize("change,match", [
    ({}, "CUDA device"), (dict(cache=torch.zeros(4, 8, 80)), "cache must be bf16"), (dict(cache=torch.zeros(4, 8, 88, dtype=bf16)), "sizes do not match"),
    (dict(q_pe=torch.zeros(2, 2, 16, dtype=bf16)), "head count mismatch"), (dict(q_pe=torch.zeros(2, 3, 16, dtype=f16)), "of the cache's type"),
    (dict(page_table=torch.zeros(2, 2, dtype=i64)), "int32"), (dict(page_table=torch.zeros(3, 2, dtype=i32)), "page_table must be"),
    (dict(lengths=torch.ones(3, dtype=i32)), "lengths must be"), (dict(lengths=torch.ones(2, dtype=i64)), "int32"),
    (dict(cache=torch.zeros(4, 8, 81, dtype=bf16)[..., :80]), "16-byte")])
def test_attention_refusals(change, match):
    _refused(match, serving.paged_mla_attention, **{**_attn_args(), **change})


def _args(good, **change):
    got = dict(good)
    got.update(change)
    return list(got.values())


def test_entry_point_codes():
    lib = native.load_library()
    norm = dict(x=FAKE, xs=256, xd=1, r=None, rs=0, w=FAKE, wd=1, rows=0, cols=256, eps=1e-6, c=FAKE, cs=256, s=FAKE, ro=None, no=None, st=None)
    f = lib.moe_rmsnorm_fp8
    assert f(*_args(norm)) == 0  # no rows: nothing to do
    assert f(*_args(norm, x=None)) == -1 and f(*_args(norm, r=FAKE)) == -1
    assert f(*_args(norm, cols=0)) == -2 and f(*_args(norm, rows=-1)) == -2 and f(*_args(norm, cs=255)) == -2
    assert f(*_args(norm, xd=3)) == -5 and f(*_args(norm, wd=2)) == -5 and f(*_args(norm, cols=32769, cs=32769)) == -5
    quant = dict(x=FAKE, xs=256, xd=1, rows=0, cols=256, c=FAKE, cs=256, s=FAKE, st=None)
    f = lib.moe_fp8_quantize_rows
    assert f(*_args(quant)) == 0 and f(*_args(quant, s=None)) == -1 and f(*_args(quant, cols=0)) == -2 and f(*_args(quant, xd=7)) == -5
    linear = dict(x=FAKE, xs=256, sx=FAKE, w=FAKE, ws=256, sw=FAKE, rows=0, outs=128, cols=256, out=FAKE, od=1, st=None)
    f = lib.moe_fp8_block_linear
    assert f(*_args(linear)) == 0 and f(*_args(linear, out=None)) == -1
    assert f(*_args(linear, outs=0)) == -2 and f(*_args(linear, xs=128)) == -2
    assert f(*_args(linear, xs=264)) == -5 and f(*_args(linear, w=ctypes.c_void_p(0x1008))) == -5 and f(*_args(linear, od=5)) == -5
    assert f(*_args(linear, rows=1 << 31)) == -5
    append = dict(kv=FAKE, ks=80, kd=1, n=FAKE, nd=1, sl=FAKE, po=FAKE, c=FAKE, s=FAKE, tr=8, ca=FAKE, cd=1, pages=4, ps=8, pst=640, rst=80,
                  q=FAKE, qs=48, qh=16, heads=3, qo=FAKE, tokens=0, latent=64, rope=16, eps=1e-6, st=None)
    f = lib.moe_paged_mla_append
    assert f(*_args(append)) == 0 and f(*_args(append, qo=None)) == -1 and f(*_args(append, sl=None)) == -1
    assert f(*_args(append, rope=15)) == -2 and f(*_args(append, pages=0)) == -2 and f(*_args(append, heads=0)) == -2
    assert f(*_args(append, pst=0)) == -5 and f(*_args(append, rst=79)) == -5  # tokens would share a row's memory
    assert f(*_args(append, cd=0)) == -5 and f(*_args(append, kd=2)) == -5 and f(*_args(append, latent=2048)) == -5
    attn = dict(ql=FAKE, qls=192, qlh=64, qp=FAKE, qps=48, qph=16, ca=FAKE, dt=1, pages=4, ps=8, pst=640, rst=80, t=FAKE, ts=2, tc=2, le=FAKE,
                batch=0, heads=3, latent=64, rope=16, sc=0.1, out=FAKE, lse=None, ws=None, wb=0, st=None)
    f = lib.moe_paged_mla_attention
    assert f(*_args(attn)) == 0 and f(*_args(attn, t=None)) == -1
    assert f(*_args(attn, tc=0)) == -2 and f(*_args(attn, sc=-1.0)) == -2 and f(*_args(attn, sc=float("nan"))) == -2
    assert f(*_args(attn, latent=520)) == -5 and f(*_args(attn, rope=72)) == -5 and f(*_args(attn, latent=60)) == -5
    assert f(*_args(attn, rst=81)) == -5 and f(*_args(attn, dt=0)) == -5 and f(*_args(attn, batch=70000)) == -5
    assert f(*_args(attn, ca=ctypes.c_void_p(0x1002))) == -5 and f(*_args(attn, ws=ctypes.c_void_p(0x1010), wb=1 << 30)) == -5
    assert f(*_args(attn, batch=2, qls=0)) == -5 and f(*_args(attn, batch=2, pst=0)) == -5
    assert f(*_args(attn, tc=1 << 20, ps=1 << 11)) == -5 and f(*_args(attn, pages=(1 << 31) - 1)) == -5  # positions and pages past 32 bits
    assert lib.moe_paged_mla_attention_workspace_bytes(2, 3, 520, 16, 2, 8) == -1
    assert lib.moe_paged_mla_attention_workspace_bytes(2, 3, 64, 16, 2, 8) >= 0


# shapes that reach every instance of the many-row linear, and the many tokens of weight streaming, on 148 SMs
LINEAR_TILES = [
    (256256, 513, 5377, 333), (256256, 2000, 2112, 1111), (256224, 257, 7109, 515), (256224, 385, 7168, 1024), (256224, 1500, 7171, 130),
    (256192, 129, 4745, 333), (256192, 2000, 5000, 1111), (256192, 256, 7680, 384), (128256, 514, 6163, 333), (128256, 600, 7168, 700),
    (128128, 100, 1003, 257), (128128, 300, 2112, 900)]


def test_linear_tiles():
    """Without a device the rule is that of 148 SMs."""
    f = native.load_library().moe_fp8_block_linear_tile
    if not torch.cuda.is_available():
        for tile, rows, outs, cols in LINEAR_TILES:
            assert f(rows, outs, cols) == tile
    assert f(1, 2112, 7168) == 16128 and f(17, 130, 257) == 32128 and f(64, 1000, 1536) == 64128
    assert f(0, 128, 128) == 0 and f(-1, 128, 128) == -2 and f(1, 0, 128) == -2 and f(1, 128, 1 << 31) == -5
