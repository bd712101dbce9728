"""What attention of a prompt in 16 bits gives, stated in 64 bits sequence by sequence: the definition that the kernel is tested against."""
import math

import torch

D = 128


def attend(q, k, v, *, scaling=None, cap=None, window=None, start=0, causal=True):
    """q [Hq, n, D] over k, v [H, m, D] in 16 bits -> out [n, Hq, D], lse [Hq, n] in 64, and how far a kernel with 32-bit sums and 16-bit weights may be off: out's rounding included."""
    dtype = q.dtype
    Hq, n, _ = q.shape
    H, m, _ = k.shape
    q, k, v = q.double(), k.double().repeat_interleave(Hq // H, dim=0), v.double().repeat_interleave(Hq // H, dim=0)
    scaling = D ** -0.5 if scaling is None else scaling
    i, j = m - n + torch.arange(n, device=q.device), torch.arange(m, device=q.device)
    seen = j[None, :] >= max(start, 0)
    seen = seen & (j <= i[:, None]) if causal else seen.expand(n, m)
    if window is not None:
        seen = seen & (j > i[:, None] - window)
    x = scaling * (q @ k.transpose(1, 2))
    size = abs(scaling) * (q.abs() @ k.abs().transpose(1, 2))             # what a sum's rounding is relative to
    if cap is not None:
        x = cap * torch.tanh(x / cap)
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, dim=-1) if m else torch.full((Hq, n), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.where(seen, torch.exp(x - torch.where(lse > -math.inf, lse, torch.zeros_like(lse))[..., None]), torch.zeros_like(x))
    # (a value that is not finite counts where it is seen alone: 0 times it is not 0)
    finite = torch.isfinite(v)
    held = torch.where(finite, v, torch.zeros_like(v))
    out, mass = w @ held, w @ held.abs()
    for h, t in (~finite).any(-1).nonzero().tolist():
        sees = seen[:, t]
        out[h, sees] += v[h, t] * torch.where(finite[h, t], 0.0, 1.0)
    # A score is off by the 128 additions of its sum and a few roundings of what it is made of, a weight by that and half a step of its 16 bits, the sums of m terms by what they
    # are; every error of one sign.  fp16: a weight below its normal numbers is off by 2^-25 where the largest is 2^8 at least.
    e32, e16 = 2.0 ** -24, torch.finfo(dtype).eps / 2
    zero = torch.zeros_like(x)
    peak = torch.where(seen, x.abs(), zero).amax(dim=-1) if m else torch.zeros_like(lse)
    size = torch.where(seen, size, zero).amax(dim=-1) if m else peak
    dx = 140 * e32 * size + 16 * e32 * (peak + (cap or 0.0) + 8)
    tol = (2 * dx + e16 + 2 * m * e32)[..., None] * mass
    if m and dtype == torch.float16:
        tol = tol + 1.01 * m * 2.0 ** -33 * held.abs().amax(dim=(1, 2))[:, None, None]
    tol = tol + (out.abs() + tol) * e16 + torch.finfo(dtype).smallest_normal * e16
    return out.transpose(0, 1), lse, tol.transpose(0, 1), dx + (m + 8) * e32


def check(got, lse, want, want_lse, tol, lse_tol):
    """got [n, Hq, D] in 16 bits and lse [Hq, n] are the definition's."""
    got, lse = got.double(), lse.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[odd].nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))
    err = (got - want).abs()
    assert bool((err <= tol)[~odd].all()), f"off by {(err / tol)[~odd].max().item()} of what it may be"
    none = want_lse == -math.inf
    assert bool((lse[none] == -math.inf).all())
    assert bool(((lse - want_lse).abs() <= lse_tol)[~none].all()), f"lse off by {((lse - want_lse).abs() / lse_tol)[~none].max().item()} of what it may be"
