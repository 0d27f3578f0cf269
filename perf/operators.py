"""The batched operators in front of the MoE layer, as cases to time and to compare.

They are the steps of a DeepSeek-V3 attention block for a batch of tokens over a paged latent cache:

  norm    s = x + residual;  y = s / sqrt(mean(s^2) + eps) * w, given as e4m3 codes with one scale for each 128 columns
  quant   the same 8-bit form of rows as they are (the attention's output before its output projection)
  linear  out = (codes * scales) . (weight codes * block scales)^T, 128-column groups against 128 x 128 blocks
  append  a token's latent row normalised and its rope part rotated into its slot of the paged cache, the queries' rope part rotated beside it
  attn    one query token per row over the pages that its table lists: softmax(scale (q_latent . c + q_pe . r)) . c

`own` false: the plain forms below, in 32 bits.  `own` true: the calls of pocketlm_b200.serving.
"""

import math

import torch

own = False

EPS = 1e-6
GROUP = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # the least amax that a group's scale is made from: an all-zero group has a scale and zero codes
LATENT, ROPE = 512, 64  # DeepSeek-V3's cache row
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode token enters a layer: latency
        {"name": "norm 1x7168", "op": "norm", "rows": 1, "cols": 7168, "type": "bf16", "residual": True, "normed": False, "pad": 0},
        # a prefill chunk enters the MoE half of a layer: codes and the router's 16-bit rows
        {"name": "norm 8192x7168", "op": "norm", "rows": 8192, "cols": 7168, "type": "bf16", "residual": True, "normed": True, "pad": 0},
        # the heads' outputs of a decode batch before the output projection
        {"name": "quant 64x16384", "op": "quant", "rows": 64, "cols": 16384, "type": "bf16", "pad": 0},
        # and of a prefill chunk
        {"name": "quant 4096x16384", "op": "quant", "rows": 4096, "cols": 16384, "type": "bf16", "pad": 0},
        # one decode token through the joined down projections of queries (1536) and cache row (576)
        {"name": "linear 1x2112x7168", "op": "linear", "rows": 1, "outs": 2112, "cols": 7168, "type": "bf16"},
        # a decode batch through the queries' up projection, 128 heads of 192
        {"name": "linear 64x24576x1536", "op": "linear", "rows": 64, "outs": 24576, "cols": 1536, "type": "bf16"},
        # a ragged prefill chunk through the output projection
        {"name": "linear 4000x7168x16384", "op": "linear", "rows": 4000, "outs": 7168, "cols": 16384, "type": "bf16"},
        # a decode batch's new cache rows, some of the batch's rows being padding
        {"name": "append 32", "op": "append", "rows": 32, "heads": 128, "type": "bf16", "page": 64, "skip": 3},
        # a prefill chunk's
        {"name": "append 4096", "op": "append", "rows": 4096, "heads": 128, "type": "bf16", "page": 64, "skip": 0},
        # one token over its own context: the work is split over the cache
        {"name": "attn 1x128 to 4096", "op": "attn", "rows": 1, "heads": 128, "longest": 4096, "type": "bf16", "page": 64, "empty": 0},
        # a rank's share of the heads, many sequences, small pages
        {"name": "attn 128x16 to 4001", "op": "attn", "rows": 128, "heads": 16, "longest": 4001, "type": "fp16", "page": 16, "empty": 2},
        # a full decode batch of long contexts
        {"name": "attn 64x128 to 8192", "op": "attn", "rows": 64, "heads": 128, "longest": 8192, "type": "bf16", "page": 64, "empty": 1},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "append", "attn"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8000), "cols": rng.choice([512, 1536, 2048, 4096, 7168, rng.randrange(1, 7168)]),
                "type": rng.choice([kind, "fp32"]), "residual": rng.random() < 0.6, "normed": rng.random() < 0.5,
                "pad": rng.choice([0, 576, rng.randrange(1, 100)])}
    if op == "quant":
        return {"op": op, "rows": _log(rng, 1, 4000), "cols": rng.choice([2048, 7168, 16384, rng.randrange(1, 8192)]),
                "type": rng.choice([kind, "fp32"]), "pad": rng.choice([0, 576, rng.randrange(1, 100)])}
    if op == "linear":
        return {"op": op, "rows": _log(rng, 1, 2000), "outs": _log(rng, 64, 8000), "cols": rng.choice([512, 1536, 2048, 7168, 16 * rng.randrange(8, 512)]),
                "type": rng.choice([kind, "fp32"])}
    if op == "append":
        rows = _log(rng, 1, 4000)
        return {"op": op, "rows": rows, "heads": rng.choice([8, 16, 32, 64, 128, rng.randrange(1, 128)]), "type": kind,
                "page": rng.choice([1, 16, 32, 48, 64, 128]), "skip": rng.randrange(0, max(1, rows // 4))}
    heads = rng.choice([8, 16, 32, 64, 128, rng.randrange(1, 128)])
    rows, longest = _log(rng, 1, 60), _log(rng, 1, 8000)
    return {"op": op, "rows": rows, "heads": heads, "longest": longest, "type": kind, "page": rng.choice([8, 16, 32, 48, 64, 128]),
            "empty": rng.randrange(0, max(1, rows // 8))}


def _lengths(case):
    """The rows' lengths: spread from a quarter of the longest up, one of them the longest, the last `empty` rows without any."""
    n = case["rows"] - case["empty"]
    got = [max(1, round(case["longest"] * (0.25 + 0.75 * ((i * 0.6180339887498949) % 1.0)))) for i in range(n)]
    got[0] = case["longest"]
    return got + [0] * case["empty"]


# ----------------------------------------------------------------- the inputs

def _quantised(t, rows):
    """Codes and scales of t's groups of `rows` x 128, for making inputs."""
    n, k = t.shape
    nb, kb = -(-n // rows), -(-k // GROUP)
    padded = torch.zeros(nb * rows, kb * GROUP, device=t.device)
    padded[:n, :k] = t
    padded = padded.view(nb, rows, kb, GROUP)
    scales = padded.abs().amax((1, 3)).clamp_min(TINY) / E4M3_MAX
    codes = (padded / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return codes.view(nb * rows, kb * GROUP)[:n, :k].to(torch.float8_e4m3fn).contiguous(), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    op, T, dt = case["op"], case["rows"], TYPES[case["type"]]
    state = {"case": case}
    if op in ("norm", "quant"):
        H = case["cols"]
        # activations with a few outlier columns, as hidden states have; the rows may be a slice of wider ones
        loud = 1 + 20 * (torch.rand(H, generator=g, device="cuda") < 0.002)
        wide = torch.zeros(T, H + case["pad"], device="cuda", dtype=dt)
        wide[:, :H] = rnd(T, H) * loud
        state["x"] = wide[:, :H]
        if op == "norm":
            state["weight"] = (1 + 0.1 * rnd(H)).to(dt)
            state["residual"] = (4 * rnd(T, H) * loud).to(dt) if case["residual"] else None
    elif op == "linear":
        state["codes"], state["scales"] = _quantised(rnd(T, case["cols"]), 1)
        state["weight"], state["scale_inv"] = _quantised(rnd(case["outs"], case["cols"]) * 0.02, GROUP)
    elif op == "append":
        page = case["page"]
        pages = -(-2 * max(T, 1024) // page)
        state["cache"] = rnd(pages, page, LATENT + ROPE).to(dt)
        state["kv"] = (3 * rnd(T, 2112)).to(dt)[:, 1536:]  # the cache row's part of the joined down projection
        state["weight"] = (1 + 0.1 * rnd(LATENT)).to(dt)
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
        if case["skip"]:
            slots[T - case["skip"]:] = -1
        state["slots"] = slots
        state["positions"] = torch.randint(0, 16384, (T,), generator=g, device="cuda")
        freq = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
        angle = torch.arange(16384, device="cuda", dtype=torch.float64)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        state["q"] = rnd(T, case["heads"], 192).to(dt)  # 128 columns without a position, then the 64 to rotate
    else:
        page = case["page"]
        lengths = _lengths(case)
        need = [-(-n // page) for n in lengths]
        total = sum(need) + 3
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
        table = torch.zeros(T, max(1, max(need)), dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        cache = torch.empty(total, page, LATENT + ROPE, device="cuda", dtype=dt)
        for i in range(0, total, 4096):
            cache[i:i + 4096] = rnd(*cache[i:i + 4096].shape)
        state["cache"], state["table"] = cache, table.cuda()
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        # scores with a spread of about 1.5 after the scale: some positions stand out, none takes all
        q = (rnd(T, case["heads"], LATENT + ROPE) * (1.5 * 192 ** 0.5 / (LATENT + ROPE) ** 0.5)).to(dt)
        state["q_latent"], state["q_pe"] = q[..., :LATENT].contiguous(), q[..., LATENT:].contiguous()
    return state


# -------------------------------------------------------------- one pass each

def _groups(y):
    T, H = y.shape
    kb = -(-H // GROUP)
    return torch.nn.functional.pad(y, (0, kb * GROUP - H)).view(T, kb, GROUP)


def _to_fp8(y):
    T, H = y.shape
    v = _groups(y)
    scales = v.abs().amax(2).clamp_min(TINY) / E4M3_MAX
    codes = (v / scales[:, :, None]).view(T, -1)[:, :H].to(torch.float8_e4m3fn)
    return codes, scales


def _wide(codes, scales, rows):
    """The 32-bit values of codes with a scale for each `rows` x 128."""
    n, k = codes.shape
    return codes.float() * scales.repeat_interleave(rows, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]


def _rotate(v, cos, sin):
    a, b = v[..., 0::2], v[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _norm(s):
    x, case = s["x"], s["case"]
    stream = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    v = stream.float()
    y = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    codes, scales = _to_fp8(y)
    out = {"codes": codes, "scales": scales}
    if s["residual"] is not None:
        out["residual"] = stream
    if case["normed"]:
        out["normed"] = y.to(x.dtype)
    return out


def _append(s):
    cache, kv = s["cache"], s["kv"].float()
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    latent = kv[:, :LATENT]
    latent = latent * torch.rsqrt(latent.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    row = torch.cat((latent, _rotate(kv[:, LATENT:], cos, sin)), 1).to(cache.dtype)
    live = s["slots"] >= 0
    cache.view(-1, LATENT + ROPE)[s["slots"][live]] = row[live]
    q = _rotate(s["q"][..., 128:].float(), cos[:, None], sin[:, None]).to(cache.dtype)
    return {"cache": cache, "q_pe": q}


def _attn(s):
    lengths, scale = s["lengths"], 192 ** -0.5
    kv = s["cache"][s["table"].long()].flatten(1, 2).float()  # every row's pages behind one another
    q = torch.cat((s["q_latent"], s["q_pe"]), 2).float()
    score = torch.matmul(q, kv.transpose(1, 2)) * scale
    live = torch.arange(kv.shape[1], device=kv.device) < lengths[:, None]
    score = score.masked_fill(~live[:, None], -math.inf)
    top = score.amax(2, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(2, keepdim=True)
    out = torch.matmul(p, kv[..., :LATENT]) / total.masked_fill(total == 0, 1.0)
    return {"out": out.to(s["q_latent"].dtype), "lse": (top + total.log())[..., 0]}


def run(state):
    op, case = state["case"]["op"], state["case"]
    if own:
        from pocketlm_b200 import serving

        if op == "norm":
            r = serving.rmsnorm_fp8(state["x"], state["weight"], residual=state["residual"], eps=EPS, return_normed=case["normed"])
            out = {"codes": r.codes, "scales": r.scales}
            if case["residual"]:
                out["residual"] = r.residual
            if case["normed"]:
                out["normed"] = r.normed
            return out
        if op == "quant":
            codes, scales = serving.quantize_fp8_rows(state["x"])
            return {"codes": codes, "scales": scales}
        if op == "linear":
            return serving.fp8_block_linear(state["codes"], state["scales"], state["weight"], state["scale_inv"], out_dtype=TYPES[case["type"]])
        if op == "append":
            q = serving.paged_mla_append(state["kv"], state["weight"], state["cache"], state["slots"], state["positions"], state["cos"],
                                         state["sin"], eps=EPS, q_pe=state["q"][..., 128:])
            return {"cache": state["cache"], "q_pe": q}
        out, lse = serving.paged_mla_attention(state["q_latent"], state["q_pe"], state["cache"], state["table"], state["lengths"],
                                               softmax_scale=192 ** -0.5, return_lse=True)
        return {"out": out, "lse": lse}
    if op == "norm":
        return _norm(state)
    if op == "quant":
        codes, scales = _to_fp8(state["x"].float())
        return {"codes": codes, "scales": scales}
    if op == "linear":
        x, w = _wide(state["codes"], state["scales"], 1), _wide(state["weight"], state["scale_inv"], GROUP)
        return torch.matmul(x, w.t()).to(TYPES[case["type"]])
    if op == "append":
        return _append(state)
    return _attn(state)


# ------------------------------------------------------ what a pass cannot avoid

def work(case):
    op, T = case["op"], case["rows"]
    size = 4 if case["type"] == "fp32" else 2
    if op in ("norm", "quant"):
        H = case["cols"]
        n = T * H
        moved = n * size + n + T * -(-H // GROUP) * 4  # rows in, codes and scales out
        if op == "norm":
            moved += H * size + (2 * n * size if case["residual"] else 0) + (n * size if case["normed"] else 0)
        return {"bytes": moved, "flops": n * (8 if op == "norm" else 3)}
    if op == "linear":
        N, K = case["outs"], case["cols"]
        kb = -(-K // GROUP)
        return {"bytes": T * K + N * K + 4 * kb * (T + -(-N // GROUP)) + T * N * size, "flops": 2 * T * N * K}
    if op == "append":
        live = T - case["skip"]
        row, q = (LATENT + ROPE) * 2, case["heads"] * ROPE * 2
        return {"bytes": live * 2 * row + T * (2 * q + 16 + ROPE * 4) + LATENT * 2, "flops": live * LATENT * 4 + (live + T * case["heads"]) * ROPE * 3}
    total, pages = sum(_lengths(case)), sum(-(-n // case["page"]) for n in _lengths(case))
    heads = case["heads"]
    moved = total * (LATENT + ROPE) * 2 + T * heads * ((2 * LATENT + ROPE) * 2 + 4) + pages * 4 + T * 4
    return {"bytes": moved, "flops": 2 * total * heads * (2 * LATENT + ROPE)}


# --------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "quant"):
        v = s["x"].double()
        out = {}
        if op == "norm":
            if s["residual"] is not None:
                v = v + s["residual"].double()
                out["residual"] = v
                v = v.to(s["x"].dtype).double()  # the norm is of the stream as it is kept
            v = v / (v.pow(2).sum(1, keepdim=True) / case["cols"] + EPS).sqrt() * s["weight"].double()
            if case["normed"]:
                out["normed"] = v
        lim = torch.stack([part.abs().amax(1) for part in v.split(GROUP, 1)], 1).clamp(min=TINY) / E4M3_MAX
        out["scales"] = lim
        out["codes"] = torch.cat([part / lim[:, i:i + 1] for i, part in enumerate(v.split(GROUP, 1))], 1)  # before the codes' rounding
        return out
    if op == "linear":
        x, w = s["codes"].double(), s["weight"].double()
        out = torch.zeros(case["rows"], case["outs"], dtype=torch.float64, device=x.device)
        rows = torch.arange(case["outs"], device=x.device) // GROUP
        for b in range(s["scales"].shape[1]):
            at = slice(b * GROUP, (b + 1) * GROUP)
            out += (x[:, at] @ w[:, at].t()) * s["scales"][:, b:b + 1].double() * s["scale_inv"][rows, b].double()
        return out
    if op == "append":
        kv, where = s["kv"].double(), s["positions"]
        c, r = kv[:, :LATENT], torch.view_as_complex(kv[:, LATENT:].reshape(-1, ROPE // 2, 2).contiguous())
        turn = torch.complex(s["cos"][where].double(), s["sin"][where].double())
        c = c / (c.pow(2).sum(1, keepdim=True) / LATENT + EPS).sqrt() * s["weight"].double()
        row = torch.cat((c, torch.view_as_real(r * turn).flatten(1)), 1)
        cache = s["cache"].double()
        page = case["page"]
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                cache[slot // page, slot % page] = row[t]
        q = torch.view_as_complex(s["q"][..., 128:].double().reshape(case["rows"], case["heads"], ROPE // 2, 2).contiguous())
        return {"cache": cache, "q_pe": torch.view_as_real(q * turn[:, None]).flatten(2)}
    out = torch.zeros(case["rows"], case["heads"], LATENT, dtype=torch.float64, device="cuda")
    lse = torch.full((case["rows"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        if n:
            rows = s["cache"][s["table"][i, :-(-n // case["page"])].long()].flatten(0, 1)[:n].double()
            score = (s["q_latent"][i].double() @ rows[:, :LATENT].t() + s["q_pe"][i].double() @ rows[:, LATENT:].t()) / math.sqrt(192)
            lse[i] = torch.logsumexp(score, 1)
            out[i] = torch.exp(score - lse[i][:, None]) @ rows[:, :LATENT]
    return {"out": out, "lse": lse}
