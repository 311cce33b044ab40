"""Linear with weights in 8-bit floating point on the fp8 matrix cores, beside ``q8.Q8Linear``.

``Q8Linear`` keeps MLX's affine codes and multiplies in fp16; ``F8Linear`` keeps e4m3 codes with one fp32 scale per
128 x 128 block of the weight, brings its input to e4m3 with one scale per row and 128 columns, and multiplies on the
fp8 matrix cores, at twice the fp16 rate and without decoding the weights. An element's error is that of e4m3 on both
sides (half a step of 2^-3 at most, 2^-4 of the value), where ``Q8Linear`` rounds weights to 1/255 of a group's range
and leaves the input alone: for weights published in this form, and where that error is bearable, as trained models'
linears mostly find it. It may stand in an ``EsmcBlock`` in the place of any of its linears.

The codes are laid out once in the order of the kernel's fragments; ``codes`` gives them back as [N, K].
"""

from __future__ import annotations

import torch
from torch import nn

from . import kernels
from .q8 import ScratchParts

BLOCK = 128
_TYPES = (torch.float16, torch.bfloat16)


class F8Linear(nn.Module):
    pair_rows = False  # (Q8Linear's gated layout: not a form of this linear)

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, device=None):
        """``codes`` [N, K] float8_e4m3fn (or their bytes, uint8), ``scales`` [ceil(N / 128), ceil(K / 128)]; K a
        multiple of 16, N of 8."""
        super().__init__()
        if codes.dim() != 2 or codes.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise ValueError(f"f8 codes: {codes.dtype} {tuple(codes.shape)} (e4m3 [N, K])")
        N, K = codes.shape
        if K % 16 or N % 8 or not K or not N or tuple(scales.shape) != (-(-N // BLOCK), -(-K // BLOCK)):
            raise ValueError(f"f8 shapes: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        q = codes.detach().view(torch.uint8).to(dev).contiguous()
        self.register_buffer("codes_packed", kernels.f8_pack_codes(q))
        self.register_buffer("scales", scales.detach().to(device=dev, dtype=torch.float32).contiguous())
        self.in_features, self.out_features = K, N

    @classmethod
    def from_float(cls, w: torch.Tensor, device=None) -> "F8Linear":
        """From weights [N, K] (torch's [out, in] layout), brought to e4m3 on the GPU block by block."""
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        q, s = kernels.f8_quantize_weight(w.detach().to(device=dev, dtype=torch.float32).contiguous())
        return cls(q, s, device=dev)

    @property
    def codes(self) -> torch.Tensor:
        """The codes [N, K], float8_e4m3fn."""
        N, K = self.out_features, self.in_features
        ng, kb = -(-N // 64), -(-K // BLOCK)
        # [piece, k block, fragment j, half, k / 32 in the block, (row / 16, row % 4), 16 k]
        p = self.codes_packed.view(ng, kb, 4, 2, 4, 4, 4, 16).permute(0, 5, 2, 6, 1, 4, 3, 7)
        return p.reshape(ng * 64, kb * BLOCK)[:N, :K].contiguous().view(torch.float8_e4m3fn)

    def dequantized(self) -> torch.Tensor:
        """W [N, K] fp32."""
        s = self.scales.repeat_interleave(BLOCK, 0)[:self.out_features]
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

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x . W^T in x's type (fp16 and bf16 as they are, others through fp16)."""
        b = self._buffers
        y = kernels.f8_linear(self._input(x), b["codes_packed"], b["scales"], self.out_features)
        if x.dim() != 2:
            y = y.reshape(*x.shape[:-1], self.out_features)
        return y if y.dtype is x.dtype else y.to(x.dtype)

    def partials(self, x: torch.Tensor) -> ScratchParts:
        """(partials [splits, M, N] fp32, splits) in the shared scratch, as ``Q8Linear.partials``: rounded to x's type,
        the sum in split order is ``forward(x)``."""
        return ScratchParts(*kernels.f8_linear_partials(self._input(x), self.codes_packed, self.scales,
                                                        self.out_features))
