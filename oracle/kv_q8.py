"""The 8-bit K/V cache in 64 bits: the format by its definition (a search over exponents, the table of the 256 codes)
and attention over the values it stands for, with the error a kernel may make on the way. Test infrastructure."""
import math
from typing import List, NamedTuple, Optional, Tuple

import torch

MIN_EXP, MAX_EXP = -64, 63


def code_values() -> torch.Tensor:
    """The 256 e4m3 codes as float64 (sign, 4 exponent bits with bias 7, 3 fraction bits; 0x7f and 0xff are NaN)."""
    v = []
    for u in range(256):
        e, f = (u >> 3) & 15, u & 7
        x = math.nan if (u & 127) == 127 else ((8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9)
        v.append(-x if u & 128 else x)
    return torch.tensor(v, dtype=torch.float64)


def values(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """Codes [..., D] and exponent bytes [...] -> float64 values."""
    table = code_values().to(codes.device)
    scale = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64, device=codes.device)
    return table[codes.view(torch.uint8).long()] * scale[byte.long()].unsqueeze(-1)


def quantise(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., D] of any float type -> (codes uint8, exponent bytes uint8): the smallest exponent under which every
    finite value fits 448, the nearest code (ties to the even one), saturating; inf and NaN become NaN."""
    x = x.double().cpu()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    e = torch.full(top.shape, MAX_EXP, dtype=torch.int64)
    for k in range(MAX_EXP - 1, MIN_EXP - 1, -1):
        e = torch.where(top <= 448.0 * 2.0 ** k, k, e)
    scale = torch.tensor([2.0 ** -k for k in range(MIN_EXP, MAX_EXP + 1)], dtype=torch.float64)[e - MIN_EXP]
    y = torch.where(fine, x * scale.unsqueeze(-1), 0.0)
    grid = code_values()[:127]                                   # 0 ... 448, ascending, code = index
    a = y.abs().clamp(max=448.0)
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = torch.where(fine, code | torch.where(torch.signbit(y), 128, 0), 127)
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


class Weights(NamedTuple):
    """How a kernel holds the softmax weights for the product with V: what a weight may be off by relative to itself, and relative to
    the largest weight (times the scale of its V row) of its query."""
    step: float
    floor: float
    adds: int           # products that enter the sums of one step of 16 keys


# One number in fp16 (half a step: 2^-11). The largest one of a query is at least 2^6 when its offset is chosen, so half of
# fp16's smallest step, 2^-25, is 2^-31 of it at the most.
FP16 = Weights(2.0 ** -11, 2.0 ** -31, 17)
# Two bf16 numbers: the first is cut off, so the rest is under 2^-7 of the weight; the second is rounded, off by 2^-8 of that rest. No
# floor (bf16 has fp32's exponents).
TWO_BF16 = Weights(2.0 ** -15, 0.0, 34)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor, scale: float, weights: Optional[Weights] = None):
    """One sequence in float64: q [m, H, D], k and v [n, kvh, D] (values), seen [m, n]. A key that a query does not see has no
    part in its row, whatever it holds. Returns (out [m, H, D], lse [m, H], err_out [m, H, D], err_lse [m, H]); the last two
    bound what a kernel may add before it rounds the output. With `weights`:
      * scores: the query loses nothing. A matrix instruction adds 16 products and the sum so far, each cut at 2^-24 of the
        largest; eight of them make a score: 8 * 17 * 2^-24, under 2^-16.9 of the sum of magnitudes;
      * a score off by d moves every weight by at most 2 d of itself (numerator and normaliser);
      * weights: their rounding, above;
      * the sums over the keys, cut in the same way, a step for every 16 keys: n / 16 * adds * 2^-24;
      * exponentials, the normaliser and the division: 2^-18.
    Without, a wider bound that also holds for query and weights as two 4-bit pieces each: 2^-18 of the query's largest value
    per product, 2^-8 of every weight, and n * 2^-22 of the largest."""
    m, H, D = q.shape
    n, kvh, _ = k.shape
    G = H // kvh
    q, k, v = q.double().view(m, kvh, G, D), k.double(), v.double()
    s = torch.einsum("mhgd,nhd->mhgn", q, k) * scale
    s = s.masked_fill(~seen[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen[:, None, None, :], torch.exp(s - lse.clamp_min(-1e300).unsqueeze(-1)), 0.0)
    any_seen = seen.any(-1)
    kk = torch.where(seen.any(0)[:, None, None], k, 0.0)
    odd = torch.isnan(v) & seen.any(0)[:, None, None]
    vv = torch.where(seen.any(0)[:, None, None] & ~odd, v, 0.0)
    out = torch.einsum("mhgn,nhd->mhgd", p, vv)
    mag = torch.einsum("mhgd,nhd->mhgn", q.abs(), kk.abs()) * abs(scale)
    hidden = ~seen[:, None, None, :]
    A = torch.einsum("mhgn,nhd->mhgd", p, vv.abs())
    top = 2.0 * vv.abs().amax(-1)                                # at least 448 * 2^e of the row
    most = (p * top.t()[None, :, None, :]).amax(-1)
    if weights is None:
        floor = q.abs().amax(-1, keepdim=True) * kk.abs().sum(-1).t()[None, :, None, :] * abs(scale)
        d = (2.0 ** -18 * floor + 2.0 ** -20 * mag).masked_fill(hidden, 0.0).amax(-1)
        err = A * (2 * d + 2.0 ** -8 + 2.0 ** -18).unsqueeze(-1) + (n * 2.0 ** -22 * most).unsqueeze(-1)
    else:
        d = (8 * 17 * 2.0 ** -24 * mag).masked_fill(hidden, 0.0).amax(-1)
        sums = -(-n // 16) * weights.adds * 2.0 ** -24
        err = A * (2 * d + weights.step + sums + 2.0 ** -18).unsqueeze(-1) + (n * weights.floor * most).unsqueeze(-1)
    hit = torch.einsum("mn,nhd->mhd", seen.double(), odd.double()) > 0
    out = out.masked_fill(hit.unsqueeze(2), math.nan)            # a NaN reaches its own dim of the queries that see it
    zero = ~any_seen[:, None, None]
    out = torch.where(zero.unsqueeze(-1), 0.0, out)
    err_lse = d + 2.0 ** -18 + 2.0 ** -22 * lse.abs().clamp(max=1e300)
    return out.reshape(m, H, D), lse.reshape(m, H), err.reshape(m, H, D), torch.where(zero, 0.0, err_lse).reshape(m, H)


def window_values(codes: torch.Tensor, scale: torch.Tensor, table: torch.Tensor, lo: int, hi: int) -> torch.Tensor:
    """Tokens [lo, hi) of one sequence through its block table: values [n, kvh, D]. codes [blocks, bs, kvh, D], scale
    [blocks, kvh, bs]."""
    bs = codes.shape[1]
    t = torch.arange(lo, hi, device=codes.device)
    blk = table[t // bs].long().clamp(0, codes.shape[0] - 1)
    return values(codes.view(torch.uint8)[blk, t % bs], scale[blk, :, t % bs])


def decode(q, codes, scales, table, lens: List[int], window_left: int, scale: float, weights: Optional[Weights] = None):
    """codes [2, ...], scales [2, ...]; q [B, H, D] -> the four tensors of attend, rows stacked."""
    return runs(q, codes, scales, table, [max(0, n - 1) for n in lens], [min(1, n) for n in lens], window_left, scale,
                one_row_each=True, weights=weights)


def runs(q, codes, scales, table, ctx: List[int], new: List[int], window_left: int, scale: float, one_row_each=False,
         weights: Optional[Weights] = None):
    """Runs of queries: sequence s owns the next new[s] rows of q, behind ctx[s] cached tokens. Tokens behind the end of the table's
    row, and those whose entry is outside the pool, are as if they were not there."""
    H, D = q.shape[1:]
    dev = q.device
    res, row = [], 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            if one_row_each:
                z = torch.zeros(1, H, D, dtype=torch.float64, device=dev)
                res.append((z, torch.full((1, H), -math.inf, dtype=torch.float64, device=dev), z, z[..., 0]))
                row += 1
            continue
        lo = 0 if window_left < 0 else max(0, c - window_left)
        hi = min(c + n, table.shape[1] * codes.shape[2])
        if hi <= lo:
            z = torch.zeros(n, H, D, dtype=torch.float64, device=dev)
            res.append((z, torch.full((n, H), -math.inf, dtype=torch.float64, device=dev), z, z[..., 0]))
            row += n
            continue
        k = window_values(codes[0], scales[0], table[s], lo, hi)
        v = window_values(codes[1], scales[1], table[s], lo, hi)
        entry = table[s][torch.arange(lo, hi, device=dev) // codes.shape[2]]
        there = ((entry >= 0) & (entry < codes.shape[1]))[None]
        for i in range(0, n, 256):
            m = min(256, n - i)
            qp = torch.arange(c + i, c + i + m, device=dev)[:, None]
            kp = torch.arange(lo, hi, device=dev)[None]
            seen = there & (kp <= qp) & ((kp >= qp - window_left) if window_left >= 0 else (kp >= 0))
            res.append(attend(q[row + i:row + i + m], k, v, seen, scale, weights))
        row += n
    return tuple(torch.cat([r[j] for r in res]) for j in range(4))
