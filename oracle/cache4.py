"""64-bit restatement of the cache in 4 bits and the attention on it, and the bound the tests hold the kernel to."""

from __future__ import annotations

import math

import torch

from .around import HALF_STEP, SMALLEST

GROUP = 64


def hold(x):
    """x [n, heads, d] -> (codes, steps, zeros), fp64, each of x's shape: s the least bf16 value, 2^-96 or more, of which 15
    reach over a group's range and 120 to its farthest value from zero; z = rint(-min / s), c = clamp(rint(x / s) + z)."""
    x = x.double()
    c, s, z = (torch.empty_like(x) for _ in range(3))
    for g in range(0, x.shape[-1], GROUP):
        v = x[..., g:g + GROUP]
        lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        least = torch.maximum(torch.maximum((hi - lo) / 15, v.abs().amax(-1, keepdim=True) / 120), torch.full_like(lo, 2.0 ** -96))
        # up to 8 binary places: 7 behind the point of a double's 52
        step = ((least.contiguous().view(torch.int64) + ((1 << 45) - 1)) >> 45 << 45).view(torch.float64)
        zero = torch.round(-lo / step)
        bad = ~torch.isfinite(v).all(-1, keepdim=True)
        step, zero = torch.where(bad, torch.full_like(step, math.nan), step), torch.where(bad, torch.zeros_like(zero), zero)
        c[..., g:g + GROUP] = torch.where(bad, torch.zeros_like(v), torch.clamp(torch.round(v / step) + zero, 0, 15))
        s[..., g:g + GROUP], z[..., g:g + GROUP] = step, zero
    return c, s, z


def attention(q, k, v, causal, scale, keep=None, u_p=2.0 ** -16):
    """(o, bound) of one sequence: q [nq, H, d] in its 16-bit type, k and v as ``hold`` gives them for its keys; ``keep`` [nk]:
    keys that may be seen at all.

    u: o's rounding. P = p s is rounded by u_p, that of two bf16 values' sum; products are exact, each sum over terms with
    16 + c and 16 + z is off by a step (2^-23) of their magnitudes' sum per addition: dS of a score, and the last term. e = 2 (dS + 2^-22 |score| + 2^-21 + (nk + 64) 2^-24) on numerator and sum, as packed attention's."""
    u, tiny = HALF_STEP[q.dtype], SMALLEST[q.dtype]
    q = q.double()
    nq, H, d = q.shape
    (kc, ks, kz), (vc, vs, vz) = k, v
    nk, Hk, _ = kc.shape
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    i, j = torch.arange(nq, device=q.device)[:, None], torch.arange(nk, device=q.device)[None]
    see = (j <= i + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool, device=q.device)
    if keep is not None:
        see = see & keep[None]
    any_seen = see.any(1)
    used = see.any(0)
    for h in range(H):
        n = h // (H // Hk)
        # what no row sees takes no part, whatever it holds
        zero = lambda t: torch.where(used[:, None], t[:, n], torch.zeros_like(t[:, n]))  # noqa: E731
        K, V = zero(ks * (kc - kz)), zero(vs * (vc - vz))
        kmag, vmag = zero(ks * ((16 + kc) + (16 + kz).abs())), zero(vs * ((16 + vc) + (16 + vz).abs()))
        sc = torch.where(see, scale * (q[:, h] @ K.t()), torch.full((nq, nk), -math.inf, dtype=torch.float64, device=q.device))
        top = torch.where(any_seen, sc.amax(1) if nk else torch.zeros(nq, device=q.device).double(), torch.zeros(nq, device=q.device).double())
        e = torch.exp(sc - top[:, None])
        l = e.sum(1, keepdim=True)
        p = torch.where(any_seen[:, None], e / torch.where(l == 0, torch.ones_like(l), l), torch.zeros_like(e))
        o[:, h] = p @ V
        ds = scale * (d + 8) * 2.0 ** -23 * (q[:, h].abs() @ kmag.t())
        ds = torch.where(see, ds, torch.zeros_like(ds)).amax(1, keepdim=True) if nk else torch.zeros(nq, 1, device=q.device)
        size = torch.where(see, sc.abs(), torch.zeros_like(sc)).amax(1, keepdim=True) if nk else torch.zeros(nq, 1, device=q.device)
        rel = 2 * (ds + 2.0 ** -22 * size + 2.0 ** -21 + (nk + 64) * 2.0 ** -24)
        A = p @ V.abs()
        # (a p below 2^-126 of the row's largest is 0)
        bound[:, h] = (u * o[:, h].abs() + (u_p + 2 * rel) * A + (2 * nk + 64) * 2.0 ** -23 * (p @ vmag)
                       + 2.0 ** -126 * V.abs().sum(0) + tiny)
    return o, bound
