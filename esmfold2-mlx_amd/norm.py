"""The residual's addition and the norm of the sum in one pass (``kernels.add_norm``), with the norm's parameters.

``h`` comes in 16 bits for any linear, or, with ``f8``, as ``f8.F8Rows``: in e4m3 as ``F8Linear`` brings its input to it,
already in the order its matrix cores take, so that neither the 16-bit rows nor the linear's own pass over them are needed.
"""

from __future__ import annotations

import torch
from torch import nn

from . import kernels
from .f8 import F8Rows


class AddNorm(nn.Module):
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, norm: str = "rms", eps: float = 1e-6, device=None):
        """``weight`` [D] and ``bias`` [D] or None, kept in fp32; ``norm``: "rms" or "layer"."""
        super().__init__()
        if norm not in ("rms", "layer") or not eps >= 0 or weight.dim() != 1 or (bias is not None and bias.shape != weight.shape):
            raise ValueError(f"AddNorm: norm={norm!r}, eps={eps}, weight {tuple(weight.shape)}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        keep = lambda t: None if t is None else t.detach().to(device=dev, dtype=torch.float32).contiguous()  # noqa: E731
        self.register_buffer("weight", keep(weight))
        self.register_buffer("bias", keep(bias))
        self.norm, self.eps = norm, float(eps)

    def forward(self, x: torch.Tensor, y: torch.Tensor | None = None, alpha: float = 1.0, *, f8: bool = False, dtype=None,
                sum_out=None, out=None):
        """(s, h): s = x + alpha * y in x's type (x itself without y) and its norm. x [..., D] fp32 or 16-bit, y and h fp16 or
        bf16 (``dtype``: h's, else y's or x's). ``f8``: h as ``F8Rows``. ``sum_out`` may be x."""
        D = self.weight.numel()
        if x.shape[-1] != D:
            raise ValueError(f"AddNorm: rows of {x.shape[-1]} values, made for {D}")
        shape = x.shape
        if x.dim() != 2:  # (views of whole rows; a copy would lose what is written to it)
            flat = lambda t: None if t is None else t.view(-1, D)  # noqa: E731
            x, y, sum_out, out = x.reshape(-1, D), None if y is None else y.reshape(-1, D), flat(sum_out), flat(out)
        kw = dict(alpha=alpha, norm=self.norm, eps=self.eps, dtype=dtype, sum_out=sum_out)
        if f8:
            if out is not None:
                raise ValueError("AddNorm: rows in e4m3 have no out")
            s, (codes, scales) = kernels.add_norm_f8(x, y, self.weight, self.bias, **kw)
            kind = dtype or (x.dtype if y is None else y.dtype)
            return s.view(shape), F8Rows(codes, scales, shape[:-1], D, kind)
        s, h = kernels.add_norm(x, y, self.weight, self.bias, out=out, **kw)
        return s.view(shape), h.view(shape)
