"""Linear with weights in 16 bits, beside ``q8.Q8Linear`` and ``f8.F8Linear``: bias, activation or gate and residual at its end.

The weights are laid out once in the order of the kernel's fragments; ``weight`` gives them back as [N, K].
"""

from __future__ import annotations

import torch
from torch import nn

from . import kernels

_TYPES = (torch.float16, torch.bfloat16)


class Linear16(nn.Module):
    pair_rows = False  # (Q8Linear's gated layout: not a form of this linear)

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, gated: bool = False, device=None):
        """``weight`` [N, K] fp16 or bf16 (multiples of 8), ``bias`` [N] (kept in fp32). ``gated``: the weight is [gate; up]
        and the linear's N / 2 outputs are act(g) u."""
        super().__init__()
        if weight.dim() != 2 or weight.dtype not in _TYPES:
            raise ValueError(f"Linear16: weight {weight.dtype} {tuple(weight.shape)} (fp16 or bf16 [N, K])")
        N, K = weight.shape
        if K % 8 or N % (16 if gated else 8) or not K or not N or (bias is not None and tuple(bias.shape) != (N,)):
            raise ValueError(f"Linear16: weight {tuple(weight.shape)} (multiples of 8, gated rows of 16), "
                             f"bias {None if bias is None else tuple(bias.shape)}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        w = weight.detach().to(dev).contiguous()
        if w.data_ptr() % 16:
            w = w.clone()
        self.register_buffer("packed", kernels.linear16_pack(w, gated))
        self.register_buffer("bias", None if bias is None else bias.detach().to(device=dev, dtype=torch.float32).contiguous())
        self.dtype, self.gated, self.rows = weight.dtype, bool(gated), N
        self.in_features, self.out_features = K, N // 2 if gated else N

    @classmethod
    def from_float(cls, w: torch.Tensor, bias: torch.Tensor | None = None, gated: bool = False, dtype=torch.float16,
                   device=None) -> "Linear16":
        """From weights [N, K] (torch's [out, in] layout), rounded to ``dtype``."""
        return cls(w.detach().to(dtype), bias, gated, device=device)

    @property
    def weight(self) -> torch.Tensor:
        """The weights [N, K]."""
        N, K = self.rows, self.in_features
        kb = -(-K // 64)
        # [piece, k block, half, fragment j, k / 8 in the half, (row / 16, row % 4), 8 k]
        p = self.packed.view(self.dtype).view(-1, kb, 2, 4, 4, 4, 4, 8).permute(0, 5, 3, 6, 1, 2, 4, 7)
        if not self.gated:  # [piece, row / 16, j, row % 4, k]
            return p.reshape(-1, kb * 64)[:N, :K].contiguous()
        p = p.reshape(-1, 4, 2, 2, 4, kb * 64)  # [piece, g, j / 2, gate or up, row % 4, k]
        return torch.cat([p[:, :, :, i].reshape(-1, kb * 64)[:N // 2, :K] for i in (0, 1)])

    def forward(self, x: torch.Tensor, activation: str | None = None, residual: torch.Tensor | None = None, alpha: float = 1.0,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """residual + alpha * act(x . W^T + bias) (gated: act(g) u), x [..., K] and residual in the weights' type."""
        K, N = self.in_features, self.out_features
        if x.shape[-1] != K or x.dtype is not self.dtype:
            raise ValueError(f"Linear16: input of {x.shape[-1]} features in {x.dtype}, takes {K} in {self.dtype}")
        shape = (*x.shape[:-1], N)
        y = kernels.linear16(_rows(x, K), self.packed, self.rows, self.bias, gated=self.gated, activation=activation,
                             residual=_residual(residual, shape), alpha=alpha, out=out)
        return y if len(shape) == 2 else y.view(shape)


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x as rows the kernel reads where they are, copied only if they must be."""
    x = x if x.dim() == 2 else x.reshape(-1, K)
    st, one = x.stride()
    if x.shape[0] and ((K > 1 and one != 1) or (x.shape[0] > 1 and (st % 8 or st < K or st > 1 << 21)) or x.data_ptr() % 16):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _residual(r, shape):
    if r is None:
        return None
    if tuple(r.shape) != tuple(shape):
        raise ValueError(f"residual {tuple(r.shape)}, the outputs are {tuple(shape)}")
    return _rows(r, shape[-1])
