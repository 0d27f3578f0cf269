"""64-bit forms of the operators of pocketlm_b200.serving, and what rounding may cost each of them."""

import torch

TINY = 2.0 ** -100
F32 = 2.0 ** -24  # half a step of fp32


def half(dtype):
    """The relative size of half a step of `dtype`."""
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half a step of the subnormals of `dtype`."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def group_scales(y):
    """max(amax, 2^-100) / 448 of each group of 128 columns of y [rows, cols]."""
    return torch.stack([g.abs().amax(1) for g in y.split(128, 1)], 1).clamp_min(TINY) / 448.0


def check_codes(codes, scales, y, rel):
    """codes * scales stand for y: the scales within `rel`, each code within half a step of y / scale."""
    want = group_scales(y)
    assert scales.shape == want.shape
    # a group that holds an infinity (a 16-bit row may): its scale is infinite, its codes NaN there and zero elsewhere
    endless = torch.isinf(want)
    assert torch.equal(torch.isinf(scales), endless)
    assert bool(((scales.double() - want).abs() <= rel * want)[~endless].all())
    s = scales.double().repeat_interleave(128, 1)[:, :y.shape[1]]
    v = y / s
    gone = endless.repeat_interleave(128, 1)[:, :y.shape[1]]
    assert torch.equal(codes.float().isnan(), torch.isinf(y)) and not codes.float()[gone & torch.isfinite(y)].any()
    off, v = (codes.double() - v).abs()[~gone], v[~gone]
    # e4m3: half a step is at most 2^-4 of a normal value, 2^-10 below 2^-6; fp32's part is `rel` of the value
    assert bool((off <= torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + v.abs() * 2 * rel).all())


def rmsnorm(x, weight, residual, eps):
    """(stream as stored, y in 64 bits)"""
    h = x if residual is None else (x.double() + residual.double()).float().to(x.dtype)
    v = h.double()
    return h, v / (v.square().mean(1, keepdim=True) + eps).sqrt() * weight.double()


def linear(codes, scales, weight, scale_inv):
    """(out, the sum of the terms' sizes) in 64 bits."""
    x = codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]
    s = scale_inv.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    w = weight.double() * s[:weight.shape[0], :weight.shape[1]]
    return x @ w.t(), x.abs() @ w.abs().t()


def rotate(v, cos, sin):
    """(rotated, the sum of the terms' sizes): pairs (2p, 2p + 1) of the last dimension."""
    a, b = v[..., 0::2], v[..., 1::2]
    out = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    size = torch.stack(((a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()), -1).flatten(-2)
    return out, size


def attention(q_latent, q_pe, cache, table, lengths, scale):
    """(out, lse, the most that rounding costs out, and lse) in 64 bits, row by row; a bad page counts as absent positions."""
    B, H, R = q_latent.shape
    half_step = half(cache.dtype)
    out = torch.zeros((B, H, R), dtype=torch.float64)
    lse = torch.full((B, H), -torch.inf, dtype=torch.float64)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    pages, page = cache.shape[:2]
    flat = cache.double().cpu()
    table, lengths = table.cpu(), lengths.cpu()
    q = torch.cat((q_latent, q_pe), 2).double().cpu()
    for b in range(B):
        n = min(max(0, int(lengths[b])), table.shape[1] * page)
        at = torch.arange(n)
        where = table[b][at // page].long() if n else at
        good = (where >= 0) & (where < pages)
        rows = flat[where[good], (at % page)[good]]
        if not len(rows):
            continue
        s = scale * (q[b] @ rows.t())
        # each score: 64-wide fp32 sums of at most (R + rope) products, a step lost per addition at worst
        ds = scale * (q[b].abs() @ rows.abs().t()).amax(1, keepdim=True) * rows.shape[1] * 2 * F32 + s.abs().amax(1, keepdim=True) * 4 * F32
        lse[b] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[b][:, None])
        c = rows[:, :R]
        out[b] = p @ c
        total = torch.exp(lse[b] - s.amax(1))[:, None]  # sum of exp(score - max), at least 1
        spread = p @ c.abs()
        # p rounded to the cache's type before its product (relative half a step, or a subnormal's half
        # step of the maximum's 1), the scores' error twice (p and the sum), fp32 sums, the result's rounding
        tol[b] = (spread * (half_step + 2 * ds + n * 2 * F32 + 2.0 ** -20) + n * least(cache.dtype) * c.abs().amax() / total
                  + half_step * out[b].abs() + least(cache.dtype))
        lse_tol[b] = ds[:, 0] + 2.0 ** -20 + 2 * F32 * lse[b].abs() + n * F32
    return out, lse, tol, lse_tol
