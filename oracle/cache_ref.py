"""The paged cache and the attention over it, in 64 bits on the CPU, from their definitions; test infrastructure only.

(The reference keeps no cache: nothing of it covers these operators - parity unpinned - and they are pinned by the definitions here alone.)"""
import math

import torch


def quantise(x):
    """Rows (..., D) -> (e4m3 values, exponents): the smallest e >= -100 with max|x| <= 448 * 2^e, x * 2^-e to the nearest of e4m3, ties to even (at e = 120 of those up to 240).

    The values come as 64-bit numbers; a row that is not finite is NaN."""
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -100, dtype=torch.int64)
    for k in range(-100, 121):
        e = torch.where(top > 448 * 2.0 ** k, k + 1, e)
    y = x * torch.exp2(-e.double())[..., None]
    step = torch.full_like(y, 2.0 ** -9)                   # the distance of e4m3 values: 2^-9 up to 2^-6, then doubled with each power of two
    for k in range(-6, 9):
        step = torch.where(y.abs() >= 2.0 ** k, 2.0 ** (k - 3), step)
    y = torch.round(y / step) * step                       # (torch.round: ties to even; the quotient is below 16, so even numbers are even mantissas)
    y = torch.where((e >= 120)[..., None], y.clamp(-240, 240), y)                              # (256 * 2^120 is no bf16 any more)
    y[~torch.isfinite(x).all(-1)] = math.nan
    return y, e


def stored(x, kind):
    """What a cache gives back for rows x."""
    if kind == "bf16":
        return x.double()
    y, e = quantise(x)
    return y * torch.exp2(e.double())[..., None]


def attend(q, k, v, scale, limits):
    """q (m, Hq, D), k, v (L, Hkv, D) -> (out, lse): row i attends keys 0 .. limits[i]; zeros and -inf where that is none.  What a row does not attend is not looked at."""
    m, hq, d = q.shape
    group = hq // k.shape[1]
    k, v = (x.double().repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))          # (Hq, L, D)
    out, lse = torch.zeros(m, hq, d, dtype=torch.float64), torch.full((hq, m), -math.inf, dtype=torch.float64)
    for i, limit in enumerate(limits):
        n = min(limit + 1, k.shape[1])
        if n <= 0:
            continue
        s = scale * (k[:, :n] @ q[i].double()[..., None])[..., 0]                             # (Hq, n)
        lse[:, i] = torch.logsumexp(s, -1)
        out[i] = (torch.softmax(s, -1)[:, None] @ v[:, :n])[:, 0]
    return out, lse
