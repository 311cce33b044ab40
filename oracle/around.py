"""64-bit restatement of what stands around the packed rows' attention: the residual's addition with the norm, the end of
a linear (bias, activation or gate, residual), and the bounds the tests hold the kernels to."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # relative to the value
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}  # below the normal range
BLOCK, TOP, FLOOR = 128, 448.0, 2.0 ** -96


def add_norm(x, y, alpha, w, b, norm, eps):
    """(s, its bound, h, its bound without a rounding) in fp64, before and after the norm of s = x + alpha y.

    s: one fp32 operation and its rounding to x's type. h: the fp32 sums over n values are off by (n + 8) 2^-24 of
    themselves, a mean's by as much of the largest value, s by 2^-24 of itself, all times 1 / sigma and w; eight more fp32
    operations on the value."""
    s = x.double() if y is None else x.double() + alpha * y.double()
    n = s.shape[1]
    m = s.mean(1, keepdim=True) if norm == "layer" else torch.zeros_like(s[:, :1])
    r = 1 / torch.sqrt(((s - m) ** 2).mean(1, keepdim=True) + eps)
    g = torch.ones(n, dtype=torch.float64, device=s.device) if w is None else w.double()
    h = (s - m) * r * g
    rel = (n + 16) * 2.0 ** -24
    bound = rel * h.abs() + 2.0 ** -24 * s.abs() * r * g.abs()
    if norm == "layer":
        bound = bound + rel * s.abs().amax(1, keepdim=True) * r * g.abs()
    if b is not None:
        h = h + b.double()
        bound = bound + 2.0 ** -24 * h.abs()
    return s, (2.0 ** -24 + HALF_STEP[x.dtype]) * s.abs() + SMALLEST[x.dtype], h, bound


def _tops(v):
    """Largest magnitude of each 8 consecutive k: [R, K] -> [R, K / 8 rounded up]."""
    R, K = v.shape
    p = torch.zeros(R, -(-K // 8) * 8, dtype=v.dtype, device=v.device)
    p[:, :K] = v.abs()
    return p.view(R, -1, 8).amax(-1)


def product16(x, w):
    """(x W^T, bound): exact products, at most K + 64 fp32 additions, each off by a step (2^-23) of the magnitudes' sum."""
    z, S = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    return z, (x.shape[1] + 64) * 2.0 ** -23 * S


def product8(xd, codes, scales):
    """The same of rows already in e4m3 (their values xd, fp64) and e4m3 weights. The matrix core aligns 8 consecutive
    products to the largest's exponent and cuts 13 places below it (measured): 7 2^-13 of the largest at most; then a step
    of fp32 for each of a block's 16 such sums and three for the scales and the sums over blocks."""
    N, K = codes.shape
    w = codes.double() * scales.double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    z, S = xd @ w.t(), xd.abs() @ w.abs().t()
    return z, 7 * 2.0 ** -13 * (_tops(xd) @ _tops(w).t()) + (16 + 3 * scales.shape[1]) * 2.0 ** -23 * S + 2.0 ** -126


def activate(z, kind):
    """(act(z), bound of the kernel's own arithmetic on exact z). An exponential's argument is off by 2^-23 of itself and the
    result by a few steps; gelu's polynomial by 0.75e-7 of z, absolute, in exact arithmetic, and by up to 8 steps (2^-23) of its
    own result in fp32, half of the 16 that the bound counts."""
    if kind is None:
        return z, torch.zeros_like(z)
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), torch.zeros_like(z)
    if kind == "gelu":
        a = z * torch.special.ndtr(z)
        return a, 0.75e-7 * z.abs() + (z * z + 16) * 2.0 ** -23 * a.abs()
    u = z if kind == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    a = z * torch.sigmoid(u)
    # (results below fp32's normal range are flushed)
    return a, (4 * u.abs().clamp_max(200) + 16) * 2.0 ** -23 * a.abs() + 2.0 ** -126 * (1 + z.abs())


def end(z, dz, bias, kind, gated, residual, alpha, dtype):
    """(y, bound) of residual + alpha act(z + bias), or alpha act(g) u; dz bounds the error of z. No activation rises faster
    than 1.13."""
    if bias is not None:
        z = z + bias.double()
        dz = dz + 2.0 ** -24 * z.abs()
    if gated:
        (g, u), (dg, du) = z.chunk(2, 1), dz.chunk(2, 1)
        a, da = activate(g, kind)
        da = da + 1.13 * dg
        y = a * u
        dy = da * u.abs() + a.abs() * du + da * du + 2.0 ** -24 * y.abs()
    else:
        y, dy = activate(z, kind)
        dy = dy + 1.13 * dz
    y, dy = alpha * y, abs(alpha) * dy + 2.0 ** -24 * (alpha * y).abs()
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -24 * y.abs()
    return y, dy + HALF_STEP[dtype] * (y.abs() + dy) + SMALLEST[dtype]
