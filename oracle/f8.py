"""64-bit restatement of the e4m3 linear with block scales: codes by the definition's fp32 steps, sums in fp64."""

from __future__ import annotations

import torch

TOP, FLOOR, BLOCK = 448.0, 2.0 ** -96, 128


def quantize_rows(x):
    """x [M, K] -> (e4m3 values [M, K] fp64, scales [M, K / 128] fp32): t = max(max |x|, 2^-96), e4m3(x (448 / t)),
    t / 448, each step rounded to fp32."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    p = torch.zeros(M, kb * BLOCK, device=x.device)
    p[:, :K] = x.float()
    p = p.view(M, kb, BLOCK)
    t = p.abs().amax(-1).clamp_min(FLOOR)
    # (tensor by tensor: torch divides by or into a number through its reciprocal, which rounds twice)
    top = torch.full_like(t, TOP)
    q = (p * (top / t)[..., None]).to(torch.float8_e4m3fn)
    return q.double().view(M, kb * BLOCK)[:, :K], t / top


def quantize_weight(w):
    """w [N, K] fp32 -> (codes float8_e4m3fn [N, K], scales [N / 128, K / 128])."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    p = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    p[:N, :K] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    t = p.abs().amax((1, 3)).clamp_min(FLOOR)
    s = t / torch.full_like(t, TOP)
    return (p / s[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous(), s


def _tops(v):
    """Largest magnitude of each 8 consecutive k: [R, K] -> [R, K / 8 rounded up]."""
    R, K = v.shape
    p = torch.zeros(R, -(-K // 8) * 8, dtype=v.dtype, device=v.device)
    p[:, :K] = v.abs()
    return p.view(R, -1, 8).amax(-1)


def linear(x, codes, scales):
    """(y, bound) in fp64. The bound: y's rounding; the matrix core's sum of 8 consecutive products, which are aligned
    to the largest's exponent and cut 13 binary places below it (measured on an MI355X, with one large and one small
    product at every distance; the 16x16x32 form does the same), 7 2^-13 of the largest product at most; a step of fp32
    (2^-23, cut or rounded) of the terms' magnitudes S for each of a block's 16 such sums, and per block three more
    for the scales' product, the FMA and the sum over splits."""
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[x.dtype]
    K, N = x.shape[1], codes.shape[0]
    q, s = (t.to(x.device) for t in quantize_rows(x.cpu()))
    xd = q * s.double().repeat_interleave(BLOCK, 1)[:, :K]
    w = codes.double() * scales.double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    y, S = xd @ w.t(), xd.abs() @ w.abs().t()
    cut = 7 * 2.0 ** -13 * (_tops(xd) @ _tops(w).t())
    return y, u * y.abs() + cut + (16 + 3 * s.shape[1]) * 2.0 ** -23 * S + 2.0 ** -24
