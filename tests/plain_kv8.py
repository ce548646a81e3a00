"""The 8-bit key/value cache and attention over it in 64 bits, from the definition: what the kernels are compared with.

A row is hd e4m3 numbers times 2^e, e the smallest whole number >= -100 with max |x| <= 448 * 2^e."""
import math

import torch

LOWEST, HIGHEST, PAGE = -100, 100, 64


def e4m3_values():
    """The 127 non-negative finite e4m3 numbers, ascending, from their bits."""
    out = []
    for code in range(127):
        exponent, mantissa = code >> 3, code & 7
        out.append(mantissa * 2.0 ** -9 if exponent == 0 else (1 + mantissa / 8) * 2.0 ** (exponent - 7))
    return torch.tensor(out, dtype=torch.float64)


def round_e4m3(y):
    """The nearest e4m3 number to every element of float64 ``y`` (ties to the even code), by looking all of them up."""
    grid = e4m3_values().to(y.device)
    mag = y.abs()
    hi = torch.searchsorted(grid, mag.contiguous()).clamp(0, 126)
    lo = (hi - 1).clamp_min(0)
    down, up = mag - grid[lo], grid[hi] - mag
    take_lo = (down < up) | ((down == up) & (lo % 2 == 0))
    return torch.copysign(torch.where(take_lo, grid[lo], grid[hi]), y)


def row_exponent(amax):
    """The smallest e >= LOWEST with amax <= 448 * 2^e, for float64 ``amax`` >= 0."""
    e = torch.full_like(amax, float(LOWEST))
    for _ in range(LOWEST, 130):
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    return e


def quantize(x):
    """(values of the codes, exponents) of the rows of float64 ``x``; exponent NaN for a row that is not one."""
    amax = x.abs().amax(-1)
    e = row_exponent(torch.nan_to_num(amax, nan=0.0, posinf=0.0))
    bad = ~torch.isfinite(x).all(-1) | (e > HIGHEST)
    e = torch.where(bad, torch.zeros_like(e), e)
    codes = round_e4m3(torch.where(bad[..., None], torch.zeros_like(x), x) / torch.exp2(e)[..., None])
    return codes, torch.where(bad, torch.full_like(e, math.nan), e)


def rotate(x, cos, sin, rot):
    """Split-half rotation of the first ``rot`` channels of float64 [N, heads, hd] by float64 tables' rows [N, rot / 2]."""
    half = rot // 2
    a, b, c, s = x[..., :half], x[..., half:rot], cos[:, None], sin[:, None]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., rot:]), -1)


def stored(codes, exps):
    """float64 rows of a pool: codes float8 [..., 64, hd] times 2^(byte - 127), NaN where the byte is 255."""
    scale = torch.exp2(exps.double() - 127)
    scale = torch.where(exps == 255, torch.full_like(scale, math.nan), scale)
    return codes.double() * scale[..., None]


def attend(q, k, v, positions, window=0):
    """(o, a): o float64 [rows, nh, hd] of float64 queries [rows, nh, hd] at ``positions`` over keys and values [nkv, length,
    hd] of one sequence, and a = sum p |v| / sum p, the scale of what rounding a weight can change.  A position whose key
    or value is not a number makes every row that sees it NaN."""
    nh, nkv = q.shape[1], k.shape[0]
    j = torch.arange(k.shape[1], device=q.device)
    sees = j[None] <= positions[:, None]
    if window:
        sees = sees & (positions[:, None] - j[None] < window)
    o, a = torch.empty_like(q), torch.empty_like(q)
    for h in range(nh):
        kk, vv = k[h // (nh // nkv)], v[h // (nh // nkv)]
        bad = (torch.isnan(kk).any(-1) | torch.isnan(vv).any(-1))
        kk, vv = torch.nan_to_num(kk), torch.nan_to_num(vv)
        s = torch.where(sees, q[:, h] @ kk.T / math.sqrt(q.shape[-1]), -math.inf)
        p = torch.softmax(s, -1)
        poison = torch.where((sees & bad[None]).any(-1), math.nan, 0.0)[:, None]
        o[:, h], a[:, h] = p @ vv + poison, p @ vv.abs()
    return o, a


def score_error(q, k, hd):
    """A bound on the error of a score in 32-bit: hd products added with a relative error of 2^-22 each (a tensor core's sums
    are cut off, not rounded), and three roundings of the result."""
    kmax = torch.nan_to_num(k).abs().amax((0, 1))
    return float((q.abs() * kmax).sum(-1).max()) / math.sqrt(hd) * (hd * 2.0 ** -22 + 2.0 ** -22)
