"""TEST INFRASTRUCTURE: the paged key-value cache in 64 bits on the CPU, position by position, and the bounds its users are
held to.  Shares no code with the package."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def quantise(x):
    """(codes as the numbers they are, biased exponents) of rows x[..., d] in float64: the least E >= 1 with max |finite| <=
    448 * 2^(E - 127), values to the nearest even multiple of e4m3's step (3 bits behind the point, least exponent -6)."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.ones(top.shape, dtype=torch.int64)
    for k in range(1, 255):
        e[top > 448.0 * 2.0 ** (k - 127)] = k + 1
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 127).double())[..., None]
    y = x.abs() / unit
    m, ex = torch.frexp(torch.where(finite, y, torch.zeros_like(y)).clamp(min=2.0 ** -6))       # y = m 2^ex, .5 <= m < 1
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), (ex - 1 - 3).double())
    code = torch.sign(x) * torch.round(y / step) * step
    return torch.where(finite, code, torch.full_like(code, math.nan)), e


def rows(pages, exps, table, seq, pos):
    """(n, heads, d) float64: rows at positions pos[i] of sequences seq[i]."""
    P = pages.shape[2]
    out = []
    for s, p in zip(seq, pos):
        page, slot = int(table[s][p // P]), p % P
        r = pages[page, :, slot].double()
        if exps is not None:
            r = r * torch.pow(torch.tensor(2.0, dtype=torch.float64), exps[page, :, slot].double() - 127)[:, None]
        out.append(r)
    return torch.stack(out)


def attend(q, k, v, scale):
    """q (Hq, d), k, v (n, Hk, d), all float64 -> out (Hq, d), lse (Hq,), and per element how far 32-bit arithmetic may be off:
    scores are off by at most dw = (d + 3) 2^-24 scale sum |q k| (d products and sums, the scale, a power of two), weights
    by a factor within exp(2 dw) (their own score and the maximum) times 1 + 2^-16 (16 bits of a weight at least take part in
    the products; exp itself, and its argument's rounding |w - max| 2^-24, which the weight's own size takes back below
    2^-24 / e), sums of n + 64 terms in any order by (n + 64) 2^-24 of the sum of magnitudes, both above and below."""
    Hq, d = q.shape
    n, Hk, _ = k.shape
    if n == 0:
        return torch.zeros_like(q), torch.full((Hq,), -math.inf, dtype=torch.float64), torch.zeros_like(q), torch.zeros(Hq, dtype=torch.float64)
    g = Hq // Hk
    kk, vv = k.repeat_interleave(g, 1).transpose(0, 1), v.repeat_interleave(g, 1).transpose(0, 1)          # (Hq, n, d)
    w = (kk * q[:, None]).sum(-1) * scale
    dw = ((d + 3) * 2.0 ** -24 * abs(scale) * (kk * q[:, None]).abs().sum(-1)).amax(-1)                    # (Hq,)
    m = w.amax(-1)
    p = torch.exp(w - m[:, None])
    total = p.sum(-1)
    out = (p[..., None] * vv).sum(1) / total[:, None]
    magnitude = (p[..., None] * vv.abs()).sum(1) / total[:, None]
    off = torch.expm1(2 * dw) + 2.0 ** -16 + 2 * (n + 64) * 2.0 ** -24
    lse = m + torch.log(total)
    return out, lse, off[:, None] * 2 * magnitude, dw + 2 * (n + 64) * 2.0 ** -24 + 2.0 ** -22 * (1 + lse.abs())


def far(got, want, bound, dtype):
    """How many times its bound the furthest element of `got` is from `want`: half a step of its type for the one rounding,
    and `bound` before it."""
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    ok = ~torch.isnan(want)
    if not ok.any():
        return 0.0
    allowed = bound + HALF_STEP[dtype] * (want.abs() + bound) + LEAST[dtype] / 2
    return float(((got - want).abs() / allowed)[ok].max())
