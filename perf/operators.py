"""The operators of the 8-bit paged K/V cache, in plain torch and as the framework's kernels.

A cache block holds, for every token and kv head, a row of D codes in e4m3 (8 bits) and one exponent
byte b, and stands for the values code * 2^(b - 127). Three operators work on it:

  cache    the new tokens' K (rotated or not) and V are quantised as they are written, and the newest tokens
           of every sequence are read back as dense tensors
  decode   attention of one query token per sequence over its window of the cache
  prefill  attention of runs of query tokens over the cache (a prompt chunk, a few tokens to verify)

`own` False: `run` computes them from elementary torch operations in 32 bits. True: `run` calls the
framework's kernels. `exact` follows the definitions in 64 bits, from the bits of the codes.
"""
import math

import torch

own = False
DEVICE = "cuda"
E_MIN, E_MAX = -64, 63          # range of a row's exponent
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------------------------------ cases
def listed():
    model = {"heads": 28, "kv_heads": 4, "dim": 128, "block": 16, "window": 4096, "dtype": "bf16"}
    shard = {**model, "heads": 7, "kv_heads": 1}
    half = {**model, "heads": 14, "kv_heads": 2, "block": 32}
    return [
        # one sequence decoding: the smallest call, all latency
        {"name": "write_1_token", "op": "cache", **model, "rotary": True, "seqs": 1, "ctx_lo": 8192, "ctx_hi": 8192,
         "new_lo": 1, "new_hi": 1, "read": 16},
        # a decode step of a full batch
        {"name": "write_256_tokens", "op": "cache", **model, "rotary": True, "seqs": 256, "ctx_lo": 8192, "ctx_hi": 8192,
         "new_lo": 1, "new_hi": 1, "read": 16},
        # one chunk of a long prompt, then read back whole
        {"name": "write_prompt_chunk", "op": "cache", **model, "rotary": True, "seqs": 1, "ctx_lo": 8192, "ctx_hi": 8192,
         "new_lo": 8192, "new_hi": 8192, "read": 8192},
        # ragged prompts of a small fp32 model with 64-dim heads, keys that come rotated already
        {"name": "write_ragged_fp32", "op": "cache", **half, "dim": 64, "dtype": "fp32", "rotary": False, "seqs": 37,
         "ctx_lo": 0, "ctx_hi": 700, "new_lo": 1, "new_hi": 300, "read": 333},
        # one sequence decoding on a full window
        {"name": "decode_1", "op": "decode", **model, "seqs": 1, "idle": 0, "len_lo": 8193, "len_hi": 8193, "spread": "even"},
        # a mixed batch: contexts from 1024 to 32768
        {"name": "decode_64_mixed", "op": "decode", **model, "seqs": 64, "idle": 0, "len_lo": 1025, "len_hi": 32769,
         "spread": "even"},
        # the full batch at 8192 tokens of context
        {"name": "decode_256", "op": "decode", **model, "seqs": 256, "idle": 0, "len_lo": 8193, "len_hi": 8193,
         "spread": "even"},
        # one GPU's share of the heads, many sequences of very different length, some rows idle
        {"name": "decode_1024_shard", "op": "decode", **shard, "seqs": 1024, "idle": 24, "len_lo": 129, "len_hi": 65537,
         "spread": "log"},
        # no window: long contexts attended whole
        {"name": "decode_4_long", "op": "decode", **model, "window": -1, "seqs": 4, "idle": 0, "len_lo": 100003,
         "len_hi": 131072, "spread": "even"},
        # several tokens per sequence to verify at once
        {"name": "verify_64x4", "op": "prefill", **model, "seqs": 64, "ctx_lo": 8190, "ctx_hi": 8190, "new_lo": 4, "new_hi": 4},
        # one chunk of a long prompt
        {"name": "prefill_chunk", "op": "prefill", **model, "seqs": 1, "ctx_lo": 8192, "ctx_hi": 8192, "new_lo": 8192,
         "new_hi": 8192},
        # ragged prompts, no window, half of the heads
        {"name": "prefill_ragged", "op": "prefill", **half, "window": -1, "seqs": 5, "ctx_lo": 0, "ctx_hi": 3001,
         "new_lo": 1, "new_hi": 2011},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    heads, kv_heads = rng.choice([(28, 4), (28, 4), (14, 2), (7, 1), (32, 4), (4, 4), (8, 2)])
    c = {"heads": heads, "kv_heads": kv_heads, "dim": 128, "block": rng.choice([16, 16, 32, 64, 128]),
         "window": rng.choice([4096, 4096, 4095, 511, rng.randint(0, 4096), -1]), "dtype": "bf16"}
    op = rng.choice(["cache", "decode", "decode", "prefill"])
    if op == "cache":
        seqs = _log_int(rng, 1, 600)
        new = _log_int(rng, 1, max(1, 8192 // seqs))
        ctx = rng.randint(0, 9000)
        c.update(op=op, seqs=seqs, ctx_lo=rng.randint(0, ctx), ctx_hi=ctx, new_lo=rng.randint(1, new), new_hi=new,
                 read=rng.randint(1, new + 40), rotary=rng.random() < 0.7, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                 dim=rng.choice([128, 128, 64]))
    elif op == "decode":
        seqs = _log_int(rng, 1, 1100)
        hi = _log_int(rng, 16, max(16, min(131072, 4 * 131072 // seqs) if c["window"] < 0 else 60000))
        c.update(op=op, seqs=seqs, idle=rng.choice([0, 0, rng.randint(0, seqs // 4)]), len_lo=rng.randint(1, hi), len_hi=hi,
                 spread=rng.choice(["even", "log"]))
        if seqs * kv_heads > 1024:           # a drawn case costs no more than the largest listed one
            c["seqs"], c["idle"] = 1024 // kv_heads, min(c["idle"], 64)
    else:
        seqs = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, max(4, 8192 // seqs))
        ctx = rng.randint(0, max(64, min(9000, 40000 // seqs)))
        c.update(op=op, seqs=seqs, ctx_lo=rng.randint(0, ctx), ctx_hi=ctx, new_lo=rng.randint(1, new), new_hi=new)
        while work(c)["flops"] > 4.5e11:
            c["new_hi"] = c["new_hi"] * 3 // 4
            c["new_lo"] = min(c["new_lo"], c["new_hi"])
    return c


def _spread(n, lo, hi, kind="even", phase=0.0):
    """n whole numbers of [lo, hi], the same for every seed; the last one is hi."""
    f = [(phase + (i + 1) * GOLDEN) % 1.0 for i in range(n)]
    v = [int(round(lo + (hi - lo) * x)) if kind == "even" else int(round(lo * (hi / lo) ** x)) for x in f]
    if n:
        v[-1] = hi
    return v


def _lengths(c):
    """(tokens cached before, new tokens, tokens afterwards) of every sequence."""
    if c["op"] == "decode":
        n = c["seqs"] - c["idle"]
        lens = _spread(n, c["len_lo"], c["len_hi"], c["spread"]) + [0] * c["idle"]
        return [max(0, x - 1) for x in lens], [min(1, x) for x in lens], lens
    ctx = _spread(c["seqs"], c["ctx_lo"], c["ctx_hi"])
    new = _spread(c["seqs"], c["new_lo"], c["new_hi"], phase=0.3)
    return ctx, new, [a + b for a, b in zip(ctx, new)]


def _first_key(c, ctx):
    """First token that a sequence's next query sees."""
    return 0 if c["window"] < 0 else max(0, ctx - c["window"])


# ------------------------------------------------------------------------------------------ inputs
def _dtype(c):
    return torch.float32 if c["dtype"] == "fp32" else torch.bfloat16


def _power(e):
    """2^e in fp32 for whole e of a normal number, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """Rows x [..., D] -> codes in e4m3 and exponent bytes: the smallest e in [E_MIN, E_MAX] with |x| <= 448 * 2^e over
    the row's finite values, codes to nearest even; what is not finite becomes NaN."""
    x = x.float()
    fine = torch.isfinite(x)
    m, k = torch.frexp(torch.where(fine, x.abs(), 0.0).amax(-1))           # amax = m * 2^k, m in [0.5, 1)
    e = torch.where(m > 0, k - 9 + (m > 0.875).int(), E_MIN).clamp(E_MIN, E_MAX)
    y = (x * _power(-e).unsqueeze(-1)).clamp(-448.0, 448.0)
    return torch.where(fine, y, float("nan")).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _dequantise(codes, byte):
    return codes.float() * _power(byte.int() - 127).unsqueeze(-1)


def _tokens(g, shape):
    """Rows of a projection: normal values, each token with a magnitude of its own."""
    x = torch.randn(shape, generator=g, device=DEVICE)
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device=DEVICE))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    ctx, new, lens = _lengths(c)
    B, H, kvh, D, bs = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["block"]
    dt = _dtype(c)
    # ---- a pool with the blocks that the case reads or writes, behind a permuted table
    if c["op"] == "cache":
        first = [min(a, max(0, n - c["read"])) // bs for a, n in zip(ctx, lens)]
    else:
        first = [_first_key(c, a) // bs for a in ctx]
    last = [-(-n // bs) for n in lens]
    nb = sum(b - a for a, b in zip(first, last)) + 3
    perm = torch.randperm(nb, generator=g, device=DEVICE).to(torch.int32)
    width = max(1, max(last))
    lo = torch.tensor(first, device=DEVICE).unsqueeze(1)
    hi = torch.tensor(last, device=DEVICE).unsqueeze(1)
    cols = torch.arange(width, device=DEVICE).unsqueeze(0)
    live = (cols >= lo) & (cols < hi)
    order = (torch.cumsum(live.flatten().long(), 0) - 1).clamp_min(0).view(B, width)
    table = torch.where(live, perm[order], -1).contiguous()
    codes, scales = [], []
    for _ in range(2):
        x, b = _quantise(_tokens(g, (nb, bs, kvh, D)))
        codes.append(x)
        scales.append(b.transpose(1, 2).contiguous())                     # [block, head, token]
        del x, b
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    s = {"case": c, "k_cache": codes[0], "v_cache": codes[1], "k_scale": scales[0], "v_scale": scales[1], "table": table,
         "lens": i32(lens), "ctx": i32(ctx), "max_len": max(lens), "max_new": max(new)}
    T = sum(new)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    s["start"] = i32(start)
    # sequence and position of every new token
    s["seq"] = torch.repeat_interleave(torch.arange(B, device=DEVICE), torch.tensor(new, device=DEVICE), output_size=T)
    s["pos"] = torch.arange(T, device=DEVICE) - s["start"].long()[s["seq"]] + s["ctx"].long()[s["seq"]]
    s["q"] = torch.randn(B if c["op"] == "decode" else T, H, D, generator=g, device=DEVICE).to(dt)
    if c["op"] == "cache":
        s["key"] = _tokens(g, (T, kvh, D)).to(dt)
        s["value"] = _tokens(g, (T, kvh, D)).to(dt)
        s["slots"] = table[s["seq"], s["pos"] // bs].long() * bs + s["pos"] % bs
        freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEVICE) / D)
        angle = torch.arange(max(lens), dtype=torch.float64, device=DEVICE).unsqueeze(1) * freq
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).to(dt)
    if c["op"] == "prefill":
        s["first"] = [_first_key(c, a) for a in ctx]
        s["keys"] = max(n - a for n, a in zip(lens, s["first"]))
        s["first"] = torch.tensor(s["first"], device=DEVICE)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _window(s, first, n):
    """Tokens first[b] ... first[b] + n - 1 of every sequence as values in fp32 [B, kvh, n, D], and which of them exist."""
    bs = s["case"]["block"]
    pos = first.long().unsqueeze(1) + torch.arange(n, device=DEVICE)
    there = pos < s["lens"].long().unsqueeze(1)
    blk = torch.gather(s["table"].long(), 1, (pos // bs).clamp_max(s["table"].shape[1] - 1)).clamp_min(0)
    off = pos % bs
    out = [_dequantise(s[x + "_cache"][blk, off], s[x + "_scale"][blk, :, off]).transpose(1, 2) for x in "kv"]
    return out[0], out[1], there


def _rotate(x, cos, sin):
    """x [T, heads, D] in fp32, cos and sin [T, 1, D/2]: the halves of a head turn together."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_cache(s):
    c = s["case"]
    k, v = s["key"].float(), s["value"].float()
    if c["rotary"]:
        cos, sin = s["cos_sin"][s["pos"]].float().unsqueeze(1).chunk(2, -1)
        s["q"].copy_(_rotate(s["q"].float(), cos, sin))
        k = _rotate(k, cos, sin)
    blk, off = s["slots"] // c["block"], s["slots"] % c["block"]
    for x, rows in (("k", k), ("v", v)):
        codes, byte = _quantise(rows)
        s[x + "_cache"].view(torch.uint8)[blk, off] = codes.view(torch.uint8)
        s[x + "_scale"][blk, :, off] = byte
    k, v, there = _window(s, (s["lens"] - c["read"]).clamp_min(0), c["read"])
    there = there[:, None, :, None]
    return {"q": s["q"], "k": torch.where(there, k, 0.0).to(_dtype(c)), "v": torch.where(there, v, 0.0).to(_dtype(c)),
            "k_codes": s["k_cache"], "v_codes": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attend(q, k, v, seen, scale):
    """q [B, kvh, R, D], k and v [B, kvh, n, D], seen [B, 1, R or 1, n] -> values [B, kvh, R, D] and log-sum-exp of the
    scores [B, kvh, R]; a row that sees nothing gives zeros and -inf."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, float("-inf"))
    m = p.amax(-1, keepdim=True)
    p.sub_(m.clamp_min(-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, torch.where(seen.any(-2).unsqueeze(-1), v, 0.0)) / torch.where(total > 0, total, 1.0)
    return out, (m + total.log()).squeeze(-1)


def _plain_decode(s):
    c = s["case"]
    B, H, kvh, D = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    n = s["max_len"] if c["window"] < 0 else min(s["max_len"], c["window"] + 1)
    first = (s["lens"] - n).clamp_min(0)
    k, v, there = _window(s, first, n)
    out, lse = _attend(s["q"].float().view(B, kvh, H // kvh, D), k, v, there[:, None, None, :], D ** -0.5)
    return {"out": out.reshape(B, H, D).to(torch.bfloat16), "lse": lse.reshape(B, H)}


def _plain_prefill(s):
    c = s["case"]
    B, H, kvh, D, n, m = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["keys"], s["max_new"]
    G = H // kvh
    k, v, there = _window(s, s["first"], n)
    at = s["pos"] - s["ctx"].long()[s["seq"]]                               # place of a token in its run
    q = torch.zeros(B, m, H, D, device=DEVICE)
    q[s["seq"], at] = s["q"].float()
    q = q.view(B, m, kvh, G, D).permute(0, 2, 3, 1, 4).reshape(B, kvh, G * m, D)
    qpos = s["ctx"].long().unsqueeze(1) + torch.arange(m, device=DEVICE)
    kpos = s["first"].unsqueeze(1) + torch.arange(n, device=DEVICE)
    seen = there.unsqueeze(1) & (kpos.unsqueeze(1) <= qpos.unsqueeze(2))
    if c["window"] >= 0:
        seen = seen & (kpos.unsqueeze(1) >= qpos.unsqueeze(2) - c["window"])
    seen = seen.repeat(1, G, 1).unsqueeze(1)                                # [B, 1, G * m, n]
    out, _ = _attend(q, k, v, seen, D ** -0.5)
    out = out.view(B, kvh, G, m, D).permute(0, 3, 1, 2, 4).reshape(B, m, H, D)
    return {"out": out[s["seq"], at].to(torch.bfloat16)}


# ------------------------------------------------------------------------------------------ the framework's kernels
def _own_cache(s):
    from spikingbrain_7b_b200 import ops
    c = s["case"]
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if c["rotary"]:
        ops.rope_kv_append_q8(s["q"], s["key"], s["value"], *cache, s["slots"], s["pos"], s["cos_sin"])
    else:
        ops.kv_append_q8(s["key"], s["value"], *cache, s["slots"])
    k, v = ops.kv_gather_q8(*cache, s["table"], s["lens"], c["read"], window_left=c["read"] - 1, dtype=_dtype(c))
    return {"q": s["q"], "k": k, "v": v, "k_codes": s["k_cache"], "v_codes": s["v_cache"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def _own_decode(s):
    from spikingbrain_7b_b200 import ops
    c = s["case"]
    lse = torch.empty(c["seqs"], c["heads"], device=DEVICE)
    out = ops.swa_decode_q8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                            window_left=c["window"], lse=lse)
    return {"out": out, "lse": lse}


def _own_prefill(s):
    from spikingbrain_7b_b200 import ops
    c = s["case"]
    return {"out": ops.swa_prefill_q8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                      s["start"], s["ctx"], s["max_new"], window_left=c["window"])}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"cache": _own_cache, "decode": _own_decode, "prefill": _own_prefill}[op](state)
    return {"cache": _plain_cache, "decode": _plain_decode, "prefill": _plain_prefill}[op](state)


# ------------------------------------------------------------------------------------------ the work of a pass
def _pairs(c, ctx, new):
    """(query, key) pairs that a run of `new` queries after `ctx` tokens sees."""
    if c["window"] < 0:
        return new * ctx + new * (new + 1) // 2
    full = c["window"] + 1
    ramp = max(0, min(new, full - ctx))              # queries that still see everything
    return ramp * ctx + ramp * (ramp + 1) // 2 + (new - ramp) * full


def work(case):
    c = dict(case)
    ctx, new, lens = _lengths(c)
    H, kvh, D = c["heads"], c["kv_heads"], c["dim"]
    es = 4 if c["dtype"] == "fp32" else 2
    row = 2 * kvh * (D + 1)                          # a token's K and V codes and exponents
    T = sum(new)
    if c["op"] == "cache":
        back = sum(min(n, c["read"]) for n in lens)
        move = T * (2 * kvh * D * es + row + 8) + back * row + c["seqs"] * c["read"] * 2 * kvh * D * es
        if c["rotary"]:
            move += T * (2 * H * D * es + D * es + 8)
        return {"bytes": move, "flops": T * (kvh * D * 8 + (6 * (H + kvh) * D // 2 if c["rotary"] else 0))}
    seen = sum(n - _first_key(c, a) for a, n in zip(ctx, lens))
    pairs = sum(_pairs(c, a, b) for a, b in zip(ctx, new))
    q = len(lens) if c["op"] == "decode" else T
    move = seen * row + 4 * (seen // c["block"]) + q * H * D * 4 + (q * H * 4 if c["op"] == "decode" else 0)
    return {"bytes": move, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(codes, byte):
    """What codes and exponent bytes stand for, from their bits: sign, 4 bits of exponent (bias 7), 3 of fraction."""
    u = codes.view(torch.uint8).long()
    e, f = (u >> 3) & 15, (u & 7).double()
    v = torch.where(e > 0, (8.0 + f) * _power64(e - 10), f * 2.0 ** -9)
    v = torch.where((u & 127) == 127, float("nan"), v)
    return torch.where(u >= 128, -v, v) * _power64(byte.long() - 127).unsqueeze(-1)


def _quantise64(x):
    """Rows in 64 bits -> (code values, exponents)."""
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2((top / 448.0).clamp_min(2.0 ** E_MIN)))
    e = torch.where(top > 448.0 * _power64(e), e + 1, e)                    # against the rounding of log2
    e = torch.where(top <= 448.0 * _power64(e - 1), e - 1, e).clamp(E_MIN, E_MAX)
    y = x * _power64(-e).unsqueeze(-1)
    step = _power64(torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 4)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0), e


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    ctx, new, lens = _lengths(c)
    H, kvh, D, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    G = H // kvh
    if c["op"] == "cache":
        q, k, v = s["q"].double(), s["key"].double(), s["value"].double()
        if c["rotary"]:
            t = s["cos_sin"].double()[s["pos"]]
            z = torch.complex(t[:, :D // 2], t[:, D // 2:]).unsqueeze(1)
            turn = lambda x: (lambda w: torch.cat([w.real, w.imag], -1))(torch.complex(x[..., :D // 2], x[..., D // 2:]) * z)  # noqa: E731
            q, k = turn(q), turn(k)
        res = {"q": q}
        for x, rows in (("k", k), ("v", v)):
            value, e = _quantise64(rows)
            stored = _values64(s[x + "_cache"], s[x + "_scale"].transpose(1, 2))          # [block, token, head, D]
            codes = _values64(s[x + "_cache"], torch.full_like(s[x + "_scale"].transpose(1, 2), 127))
            byte = s[x + "_scale"].clone()
            blk, off = s["slots"] // bs, s["slots"] % bs
            stored[blk, off] = value * _power64(e).unsqueeze(-1)
            codes[blk, off] = value
            byte[blk, :, off] = (e + 127).to(torch.uint8)
            dense = torch.zeros(c["seqs"], kvh, c["read"], D, dtype=torch.float64, device=DEVICE)
            for b, n in enumerate(lens):
                m = min(n, c["read"])
                at = torch.arange(n - m, n, device=DEVICE)
                dense[b, :, :m] = stored[s["table"][b, at // bs].long(), at % bs].transpose(0, 1)
            res.update({x: dense, x + "_codes": codes, x + "_scale": byte})
        return res
    if 4.0 * sum(_pairs(c, a, b) for a, b in zip(ctx, new)) * H * D > 4e12:
        return None
    scale = 1.0 / math.sqrt(D)
    rows = c["seqs"] if c["op"] == "decode" else sum(new)
    out = torch.zeros(rows, H, D, dtype=torch.float64, device=DEVICE)
    lse = torch.full((rows, H), -math.inf, dtype=torch.float64, device=DEVICE)
    row = 0
    for b, (a, n) in enumerate(zip(ctx, new)):
        r0 = b if c["op"] == "decode" else row
        row += n
        for i in range(0, n, 512):                                          # runs of queries
            m = min(512, n - i)
            lo, hi = _first_key(c, a + i), a + i + m
            at = torch.arange(lo, hi, device=DEVICE)
            blk = s["table"][b, at // bs].long()
            k = _values64(s["k_cache"][blk, at % bs], s["k_scale"][blk, :, at % bs])     # [n, kvh, D]
            v = _values64(s["v_cache"][blk, at % bs], s["v_scale"][blk, :, at % bs])
            q = s["q"][r0 + i:r0 + i + m].double().view(m, kvh, G, D)
            w = torch.einsum("mhgd,nhd->hgmn", q, k) * scale
            qpos = torch.arange(a + i, a + i + m, device=DEVICE).unsqueeze(1)
            hidden = at > qpos
            if c["window"] >= 0:
                hidden = hidden | (at < qpos - c["window"])
            w = w.masked_fill(hidden, -math.inf)
            lse[r0 + i:r0 + i + m] = torch.logsumexp(w, -1).permute(2, 0, 1).reshape(m, H)
            out[r0 + i:r0 + i + m] = torch.einsum("hgmn,nhd->mhgd", torch.softmax(w, -1), v).reshape(m, H, D)
    return {"out": out, "lse": lse} if c["op"] == "decode" else {"out": out}
