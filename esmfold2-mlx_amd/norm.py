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
        w, b = self._buffers["weight"], self._buffers["bias"]
        shape = x.shape
        D = shape[-1]
        if D != w.numel():
            raise ValueError(f"AddNorm: rows of {D} values, made for {w.numel()}")
        if f8 and out is not None:
            raise ValueError("AddNorm: rows in e4m3 have no out")
        flat = len(shape) == 2
        if not flat:  # (views of whole rows; a copy would lose what is written to it)
            for name, t in (("y", y), ("sum_out", sum_out), ("out", out)):
                if t is not None and t.shape != shape:
                    raise ValueError(f"AddNorm: {name} {tuple(t.shape)}, x is {tuple(shape)}")
            view = lambda t: None if t is None else t.view(-1, D)  # noqa: E731
            x, y, sum_out, out = x.reshape(-1, D), None if y is None else y.reshape(-1, D), view(sum_out), view(out)
        s, h = kernels._add_norm("add_norm", x, y, w, b, alpha, self.norm, self.eps, dtype, sum_out, out, f8)
        if f8:
            h = F8Rows(*h, shape[:-1], D, dtype or (x.dtype if y is None else y.dtype))
        if flat:
            return s, h
        return s.view(shape), h if f8 else h.view(shape)
