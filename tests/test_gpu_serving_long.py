"""Calls that last longer than the limit of any one wait (2 s): a wait is bounded by the progress that it waits for,
not by the call, so a call that moves on is complete and leaves no error."""

import math

import pytest
import torch

import serving_oracle as oracle
from pocketlm_b200 import native, serving

pytestmark = pytest.mark.gpu

LIMIT_MS = 2000.0


@pytest.fixture(autouse=True)
def _memory_goes_back(cuda_device):
    """The tests behind these start processes of their own, which need the memory."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _timed(call):
    """What call() gives and the milliseconds that it takes on the device."""
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = call()
    end.record()
    torch.cuda.synchronize()
    return got, start.elapsed_time(end)


def _error_word():
    return native.load_library().moe_b200_device_error(native._stream())


def _room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


def test_attention_longer_than_a_wait():
    """Rows that walk the same sixteen pages over and over: the attention over the pages once, its lse higher by log(turns)."""
    _room(8)
    heads, page, cols, turns = 8, 64, 8192, 512
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.randn(16, page, 576, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(1, heads, 576, generator=g, device="cuda").to(torch.bfloat16)
    once = torch.arange(16, dtype=torch.int32, device="cuda")[None]
    table = once.repeat(1, turns)
    assert table.shape[1] == cols

    def call(batch):
        lengths = torch.full((batch,), cols * page, dtype=torch.int32, device="cuda")
        rows = q.expand(batch, -1, -1)
        return serving.paged_mla_attention(rows[..., :512], rows[..., 512:], cache, table.expand(batch, -1), lengths,
                                           softmax_scale=576 ** -0.5, return_lse=True)

    call(74)
    _error_word()
    _, ms = _timed(lambda: call(1024))
    batch = min(65535, math.ceil(1024 * 1.3 * LIMIT_MS / ms))
    (out, lse), ms = _timed(lambda: call(batch))
    print(f"{batch} rows: {ms:.0f} ms")
    assert ms > LIMIT_MS  # a shorter call shows nothing
    assert _error_word() == 0
    n = torch.tensor([16 * page], dtype=torch.int32, device="cuda")
    want, want_lse, tol, lse_tol = oracle.attention(q[..., :512], q[..., 512:], cache, once, n, 576 ** -0.5)
    # the turns add 2^9 times as many terms: a tile is one more addition to a thread's sum of probabilities, and eight to the
    # result (128 positions, 16 at a time), each a step at worst of what is there, at most the largest |value| times the sum
    tiles = cols * page // 128
    more, values = tiles * 2 * oracle.F32, float(cache.abs().max())
    want, tol, want_lse, lse_tol = (t.cuda() for t in (want, tol, want_lse, lse_tol))
    off, lse_off = (out.double() - want).abs(), (lse.double() - want_lse - math.log(turns)).abs()
    assert bool((off <= tol + 9 * more * values).all())
    assert bool((lse_off <= lse_tol + more + 2 * oracle.F32 * math.log(turns)).all())


def test_linear_longer_than_a_wait():
    """Codes and weight in the same memory, all 1, and scales that add up to 1: outputs of 1."""
    _room(72)
    cols, most = 409600, 98304
    codes = torch.full((most, cols), 0x38, dtype=torch.uint8, device="cuda")  # 1 in e4m3
    blocks = cols // 128
    scales = torch.full((most, blocks), 2.0 ** -7, device="cuda")
    scale_inv = torch.full((most // 128, blocks), 1 / blocks, device="cuda")

    def call(rows):
        return serving.fp8_block_linear(codes[:rows], scales[:rows], codes, scale_inv)

    _error_word()
    _, ms = _timed(lambda: call(8192))
    rows = min(most, math.ceil(32 * 1.3 * LIMIT_MS / ms) * 256)  # whole tiles of a pair of CTAs
    out, ms = _timed(lambda: call(rows))
    print(f"{rows} rows: {ms:.0f} ms")
    assert ms > LIMIT_MS  # a shorter call shows nothing
    assert native.load_library().moe_fp8_block_linear_tile(rows, most, cols) // 1000 == 256  # a pair's tiles
    assert _error_word() == 0
    # 3200 groups whose sums are 128, exactly, times 2^-7 / 3200, rounded, added in fp32 to at most 1; then bf16's rounding
    assert bool(((out.float() - 1).abs() <= blocks * 2 * oracle.F32 + oracle.half(torch.bfloat16)).all())
