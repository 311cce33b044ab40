"""64-bit CPU restatement of the operators over packed rows (attention within sequences, the norm of queries and keys
with their rotation), and the error bounds the tests hold the kernels to."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # a rounding, relative to the value
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # and below the normal range, absolute
SMALLEST_P = {torch.float16: 2.0 ** -36, torch.bfloat16: 2.0 ** -126}  # the same of a probability, of the row's largest


def attention(q, k, v, cu_q, cu_k, causal, scale):
    """(o, bound) in fp64: rows of no sequence NaN; bound on |kernel - o| by arithmetic, element by element.

    With u the half step of the type, A = sum_j p_j |v_j| / l and e the relative error of a p:
      o's rounding u |o|; each p's rounding u (and an absolute one: at most SMALLEST_P / l each, l >= 1, as fp16's p
      are kept 2^11 times as large and bf16's are 0 below 2^-126); e = 2 dS + 2^-21 with dS = scale (d + 2) 2^-24 sum |q| |k| the fp32 score's error,
      2^-22 |scale s| the exponent argument's (a product and an FMA at the size of m c); sums over nk keys and
      the rescalings: (nk + 64) 2^-24; each of them on the numerator and the sum: twice."""
    u, tiny, tiny_p = HALF_STEP[q.dtype], SMALLEST[q.dtype], SMALLEST_P[q.dtype]
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    Tq, H, d = q.shape
    G = H // k.shape[1]
    o = torch.full((Tq, H, d), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for s in range(len(cu_q) - 1):
        a, b, ka, kb = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        nq, nk = b - a, kb - ka
        for h in range(H):
            x, y, z = q[a:b, h], k[ka:kb, h // G], v[ka:kb, h // G]
            see = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                see = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + nk - nq
            for i in range(nq):  # unseen keys take no part at all
                w = see[i]
                if not w.any():
                    o[a + i, h] = 0
                    continue
                sc = (y[w] @ x[i]) * scale
                e = torch.exp(sc - sc.max())
                l = e.sum()
                o[a + i, h] = (e / l) @ z[w]
                A = (e / l) @ z[w].abs()
                ds = scale * (d + 2) * 2.0 ** -24 * float((y[w].abs() @ x[i].abs()).max())
                rel = 2 * (ds + 2.0 ** -22 * float(sc.abs().max()) + 2.0 ** -21 + (int(w.sum()) + 64) * 2.0 ** -24)
                bound[a + i, h] = (u * o[a + i, h].abs() + (u + 2 * rel) * A + tiny_p * z[w].abs().sum(0) + tiny)
    return o, bound


def norm_rope(x, w, pos, freq, gain, rot, interleaved, norm, over, eps):
    """(y, bound) in fp64. The bound: y's rounding; the statistics' fp32 sums, (n + 8) 2^-24 relative, and for a
    layer norm the mean's, as much of the largest value times its scale; the hardware's sine and cosine, 2^-18
    absolute; six fp32 operations on the way."""
    u, tiny = HALF_STEP[x.dtype], SMALLEST[x.dtype]
    x = x.detach().cpu().double()
    T, H, d = x.shape
    y, rel, off = x.clone(), 0.0, torch.zeros(T, 1, 1, dtype=torch.float64)
    if norm:
        dims = (1, 2) if over == "row" else (2,)
        n = H * d if over == "row" else d
        top = x.abs().amax(dims, keepdim=True)
        if norm == "layer":
            y = y - y.mean(dims, keepdim=True)
        r = 1 / torch.sqrt((y ** 2).mean(dims, keepdim=True) + eps)
        y = y * r
        g = torch.ones(1, d, dtype=torch.float64)
        if w is not None:
            g = w.detach().cpu().double().view(-1, d)
        y = y * g
        rel = (n + 8) * 2.0 ** -24
        if norm == "layer":
            off = (n + 8) * 2.0 ** -24 * top * r * g.abs().amax()
    slack = rel * y.abs() + off
    angle = pos.detach().cpu().double()[:, None] * freq.detach().cpu().double()
    c, s = (gain * torch.cos(angle))[:, None], (gain * torch.sin(angle))[:, None]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, bound = y.clone(), slack.clone().expand_as(y).clone()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    size, both = y[..., a].abs() + y[..., b].abs(), slack.expand_as(y)[..., a] + slack.expand_as(y)[..., b]
    turned = (2.0 ** -18 + 6 * 2.0 ** -24) * abs(gain) * size + abs(gain) * both
    bound[..., a], bound[..., b] = turned, turned
    return out, u * out.abs() + bound + 6 * 2.0 ** -24 * out.abs() + tiny
