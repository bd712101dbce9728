"""What a paged 8-bit cache holds and what its attention gives, stated in 64 bits row by row: the definition that the kernels are tested against."""
import math

import torch

BLOCK, D = 64, 128
TOP = {"int8": 127.0, "e4m3": 448.0}
LARGEST = {torch.float16: 65504.0, torch.bfloat16: 3.3895313892515355e38}


def finite(x):
    return torch.where(torch.isfinite(x), x, torch.zeros_like(x))


def scale_of(a, top):
    """The smallest number of 8 significant bits that is not below a / top (a: 64-bit numbers), 2^-100 at least; 0 for 0."""
    m, e = torch.frexp(a / top)
    return torch.where(a > 0, (torch.ceil(m * 256) * 2.0 ** (e - 8).double()).clamp(min=2.0 ** -100), torch.zeros_like(a))


def held(x, kind):
    """x [H, n, D] in 16 bits -> what the cache holds of it in 64: full blocks as codes times scales, the rest as it is."""
    x = finite(x).double()
    H, n, _ = x.shape
    full = n // BLOCK * BLOCK
    b = x[:, :full].reshape(H, full // BLOCK, BLOCK, D)
    s = scale_of(b.abs().amax(dim=(-1, -2), keepdim=True), TOP[kind]) if full else torch.zeros(H, 0, 1, 1, dtype=torch.float64)
    y = b / torch.where(s > 0, s, torch.ones_like(s))
    if kind == "e4m3":
        step = 2.0 ** (torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4).double()
        y = (y / step).round() * step
    else:
        y = y.round()
    return torch.cat([(y * s).reshape(H, full, D), x[:, full:]], dim=1)


def to_type(x, dtype):
    """64 bits to 16, values behind the type's end at its end."""
    return x.clamp(-LARGEST[dtype], LARGEST[dtype]).to(dtype)


def cut(x, n, kind):
    """The tokens that are left of x [H, m, D] (16 bits) when a row is cut to n: those of a full block that is cut are, from then on, the values it held."""
    m = x.shape[1]
    if n >= m:
        return x
    if n // BLOCK == m // BLOCK:
        return x[:, :n]
    keep = n // BLOCK * BLOCK
    return torch.cat([x[:, :keep], to_type(held(x, kind)[:, keep:n], x.dtype)], dim=1)


def attend(q, k, v, *, scaling=None, cap=None, slopes=None, window=None, prefix=None, starts=None):
    """q [Hq, n, D] of a row's newest n tokens, k, v [H, m, D] in 64 bits -> out [n, Hq, D], lse [Hq, n], and how far a kernel with 32-bit sums and 16-bit
    weights may be off: (out [n, Hq, D] without the rounding of the result, lse [Hq, n])."""
    Hq, n, _ = q.shape
    H, m, _ = k.shape
    q = q.double()
    k, v = (x.repeat_interleave(Hq // H, dim=0) for x in (k, v))
    scaling = D ** -0.5 if scaling is None else scaling
    x = scaling * (q @ k.transpose(1, 2))
    size = abs(scaling) * (q.abs() @ k.abs().transpose(1, 2))             # what a sum's rounding is relative to
    if cap is not None:
        x = cap * torch.tanh(x / cap)
    i = m - n + torch.arange(n)
    j = torch.arange(m)
    away = (i[:, None] - j).abs().double()
    if slopes is not None:
        x = x - slopes.double()[:, None, None] * away
    lo = torch.zeros(n, dtype=torch.int64) if starts is None else starts.long().expand(n)
    if window is not None:
        lo = torch.maximum(lo, i - window + 1)
    hi = i + 1 if prefix is None else (i + 1).clamp(min=prefix)
    seen = (j >= lo[:, None]) & (j < hi.clamp(max=m)[:, None]) & (i >= 0)[:, None]
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, dim=-1) if m else torch.full((Hq, n), -math.inf, dtype=torch.float64)
    w = torch.where(seen, torch.exp(x - torch.where(lse > -math.inf, lse, torch.zeros_like(lse))[..., None]), torch.zeros_like(x))
    out, mass = w @ v, w @ v.abs()
    # a score is off by the 128 additions of its sum and a few roundings of what it is made of, a weight by that and, in 16 bits, half a step of
    # fp16, the sum of the weights by what they are; both bounds are the worst case, every error of one sign
    e32, e16 = 2.0 ** -24, 2.0 ** -11
    peak = torch.where(seen, x.abs(), torch.zeros_like(x)).amax(dim=-1) if m else torch.zeros(Hq, n, dtype=torch.float64)
    size = torch.where(seen, size, torch.zeros_like(size)).amax(dim=-1) if m else peak
    dx = 140 * e32 * size + 16 * e32 * (peak + (cap or 0.0) + 8)
    tol = (2 * dx + e16 + 2 * m * e32)[..., None] * mass
    # weights below fp16's normal numbers are off by 2^-25 at most, half a step, where the sums' unit makes the largest value 127 to 128 and a weight
    # of one (or more, never less: the sum is at least that) 2^7: a token adds 2^-25 * 2^-7 of the largest value
    if m:
        tol = tol + 1.01 * m * 2.0 ** -32 * v.abs().amax(dim=(1, 2))[:, None, None]
    return out.transpose(0, 1), lse, tol.transpose(0, 1), dx + (m + 8) * e32
