"""Linear with weights in 8-bit floating point on the fp8 matrix cores, beside ``q8.Q8Linear``.

``Q8Linear`` keeps MLX's affine codes and multiplies in fp16; ``F8Linear`` keeps e4m3 codes with one fp32 scale per
128 x 128 block of the weight, brings its input to e4m3 with one scale per row and 128 columns, and multiplies on the
fp8 matrix cores, at twice the fp16 rate and without decoding the weights. An element's error is that of e4m3 on both
sides (half a step of 2^-3 at most, 2^-4 of the value), where ``Q8Linear`` rounds weights to 1/255 of a group's range
and leaves the input alone: for weights published in this form, and where that error is bearable, as trained models'
linears mostly find it. It may stand in an ``EsmcBlock`` in the place of any of its linears.

The codes are laid out once in the order of the kernel's fragments; ``codes`` gives them back as [N, K].

Its input may already be in e4m3 (``F8Rows``, from ``norm.AddNorm``), and its end may add a bias, apply an activation or a
gate and add a residual, as ``linear.Linear16``'s.
"""

from __future__ import annotations

import torch
from torch import nn

from . import kernels
from .linear import _residual
from .q8 import ScratchParts

BLOCK = 128
_TYPES = (torch.float16, torch.bfloat16)


class F8Rows:
    """Rows [..., K] in e4m3, with a scale per row and 128 columns, in the order ``F8Linear`` takes (``kernels.add_norm_f8``)."""

    def __init__(self, packed: torch.Tensor, packed_scales: torch.Tensor, shape, features: int, dtype: torch.dtype):
        self.packed, self.packed_scales, self.shape = packed, packed_scales, shape
        self.rows = shape[0] if len(shape) == 1 else torch.Size(shape).numel()
        self.features, self.dtype = features, dtype  # dtype: of a linear's outputs

    @property
    def codes(self) -> torch.Tensor:
        """The codes [rows, K], float8_e4m3fn."""
        mb, kb = -(-self.rows // 16), -(-self.features // BLOCK)
        # [row / 16, k block, half, k / 32 in the block, row % 16, 16 k]
        p = self.packed.view(mb, kb, 2, 4, 16, 16).permute(0, 4, 1, 3, 2, 5)
        return p.reshape(mb * 16, kb * BLOCK)[:self.rows, :self.features].contiguous().view(torch.float8_e4m3fn)

    @property
    def scales(self) -> torch.Tensor:
        """The scales [rows, ceil(K / 128)] fp32."""
        mp, kb = -(-self.rows // 16) * 16, -(-self.features // BLOCK)
        return self.packed_scales[:kb * mp].view(kb, mp)[:, :self.rows].t().contiguous()

    def dequantized(self) -> torch.Tensor:
        """The values [..., K] fp32."""
        s = self.scales.repeat_interleave(BLOCK, 1)[:, :self.features]
        return (self.codes.float() * s).view(*self.shape, self.features)


def _gated_rows(N: int, device) -> torch.Tensor:
    """The order of a [gate; up] weight's rows in which a gate and its up value meet in the kernel: rows 16 g + 4 j + e of a
    piece of 64 are, for even j, the gates, for odd j the up values of outputs 8 g + 4 (j / 2) + e of the piece's 32."""
    o = torch.arange(N // 2, device=device).view(-1, 4, 2, 1, 4)  # [piece, g, j / 2, gate or up, e]
    return torch.cat([o, o + N // 2], 3).reshape(-1)


class F8Linear(nn.Module):
    pair_rows = False  # (Q8Linear's gated layout: not a form of this linear)

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, device=None, bias: torch.Tensor | None = None,
                 gated: bool = False):
        """``codes`` [N, K] float8_e4m3fn (or their bytes, uint8), ``scales`` [ceil(N / 128), ceil(K / 128)]; K a
        multiple of 16, N of 8. ``bias`` [N] (kept in fp32). ``gated``: the weight is [gate; up], N a multiple of 64, and the
        linear's N / 2 outputs are act(g) u."""
        super().__init__()
        if codes.dim() != 2 or codes.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise ValueError(f"f8 codes: {codes.dtype} {tuple(codes.shape)} (e4m3 [N, K])")
        N, K = codes.shape
        if K % 16 or N % 8 or not K or not N or tuple(scales.shape) != (-(-N // BLOCK), -(-K // BLOCK)):
            raise ValueError(f"f8 shapes: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
        if (gated and N % 64) or (bias is not None and tuple(bias.shape) != (N,)):
            raise ValueError(f"f8 shapes: {N} rows, gated {gated} (a multiple of 64), bias {None if bias is None else tuple(bias.shape)}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        q = codes.detach().view(torch.uint8).to(dev).contiguous()
        if gated:
            q = q[_gated_rows(N, dev)]
        self.register_buffer("codes_packed", kernels.f8_pack_codes(q))
        self.register_buffer("scales", scales.detach().to(device=dev, dtype=torch.float32).contiguous())
        if bias is not None:  # (no buffer without one: state dicts stay as they were)
            self.register_buffer("bias", bias.detach().to(device=dev, dtype=torch.float32).contiguous())
        self.in_features, self.out_features, self.gated, self.rows = K, N // 2 if gated else N, bool(gated), N

    @classmethod
    def from_float(cls, w: torch.Tensor, device=None, bias: torch.Tensor | None = None, gated: bool = False) -> "F8Linear":
        """From weights [N, K] (torch's [out, in] layout), brought to e4m3 on the GPU block by block."""
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        q, s = kernels.f8_quantize_weight(w.detach().to(device=dev, dtype=torch.float32).contiguous())
        return cls(q, s, device=dev, bias=bias, gated=gated)

    @property
    def codes(self) -> torch.Tensor:
        """The codes [N, K], float8_e4m3fn."""
        N, K = self.rows, self.in_features
        ng, kb = -(-N // 64), -(-K // BLOCK)
        # [piece, k block, fragment j, half, k / 32 in the block, (row / 16, row % 4), 16 k]
        p = self.codes_packed.view(ng, kb, 4, 2, 4, 4, 4, 16).permute(0, 5, 2, 6, 1, 4, 3, 7)
        q = p.reshape(ng * 64, kb * BLOCK)[:N, :K].contiguous()
        if self.gated:
            q = torch.empty_like(q).index_copy_(0, _gated_rows(N, q.device), q)
        return q.view(torch.float8_e4m3fn)

    def dequantized(self) -> torch.Tensor:
        """W [N, K] fp32."""
        s = self.scales.repeat_interleave(BLOCK, 0)[:self.rows]
        return self.codes.float() * s.repeat_interleave(BLOCK, 1)[:, :self.in_features]

    def _input(self, x: torch.Tensor) -> torch.Tensor:
        """x as rows the kernel reads where they are, copied only if they must be."""
        K = self.in_features
        if x.shape[-1] != K:
            raise ValueError(f"F8Linear: input of {x.shape[-1]} features, takes {K}")
        x2 = x if x.dim() == 2 else x.reshape(-1, K)
        if x2.dtype not in _TYPES:
            x2 = x2.to(torch.float16)
        st, one = x2.stride()
        if one != 1 or st % 8 or st < K or x2.data_ptr() % 16:
            x2 = x2.contiguous()
            if x2.data_ptr() % 16:
                x2 = x2.clone()
        return x2

    def forward(self, x, activation: str | None = None, residual: torch.Tensor | None = None, alpha: float = 1.0) -> torch.Tensor:
        """x . W^T in x's type (fp16 and bf16 as they are, others through fp16); with an end, residual + alpha * act(x . W^T +
        bias) (gated: act(g) u), the residual in the outputs' 16-bit type. x may be ``F8Rows``."""
        b = self._buffers
        bias = b.get("bias")
        if type(x) is not F8Rows and not (self.gated or bias is not None or activation is not None or residual is not None
                                          or alpha != 1.0):
            y = kernels.f8_linear(self._input(x), b["codes_packed"], b["scales"], self.out_features)
            if x.dim() != 2:
                y = y.reshape(*x.shape[:-1], self.out_features)
            return y if y.dtype is x.dtype else y.to(x.dtype)
        kw = dict(gated=self.gated, activation=activation, alpha=alpha)
        if type(x) is F8Rows:
            if x.features != self.in_features:
                raise ValueError(f"F8Linear: input of {x.features} features, takes {self.in_features}")
            shape, dtype = (*x.shape, self.out_features), x.dtype
            y = kernels.f8_linear_end(None, b["codes_packed"], b["scales"], self.rows, bias, residual=_residual(residual, shape),
                                      rows=(x.packed, x.packed_scales, x.rows, x.features), dtype=dtype, **kw)
        else:
            shape, dtype = (*x.shape[:-1], self.out_features), x.dtype
            y = kernels.f8_linear_end(self._input(x), b["codes_packed"], b["scales"], self.rows, bias,
                                      residual=_residual(residual, shape), **kw)
        y = y if len(shape) == 2 else y.view(shape)
        return y if y.dtype is dtype else y.to(dtype)

    def partials(self, x: torch.Tensor) -> ScratchParts:
        """(partials [splits, M, N] fp32, splits) in the shared scratch, as ``Q8Linear.partials``: rounded to x's type,
        the sum in split order is ``forward(x)``."""
        if self.gated or self._buffers.get("bias") is not None:
            raise ValueError("F8Linear.partials: a bias or a gate comes after the partials' sum")
        return ScratchParts(*kernels.f8_linear_partials(self._input(x), self.codes_packed, self.scales,
                                                        self.out_features))
