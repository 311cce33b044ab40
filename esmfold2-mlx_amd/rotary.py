"""Rotary positions for ``kernels.qk_norm_rope``: the angle of each pair per position, and its stretching for
contexts longer than the trained one.

The language model of ``esmc`` turns all 64 values of a head in the half layout at base 10000; ``Rotary`` covers what
other models do: pairs side by side, part of each head, another base, and four ways of stretching:

* ``linear``: every angle divided by ``factor``;
* ``ntk``: the base multiplied by factor^(rot / (rot - 2)), which stretches the slowest pair by ``factor`` and leaves
  the fastest;
* ``bands``: by the turns a pair makes within the trained ``context``: fewer than ``low`` (1) divided by ``factor``,
  more than ``high`` (4) kept, linear in the turns between;
* ``yarn``: linear in the pair's index between the pair of ``fast`` (32) turns, kept, and the one of ``slow`` (1),
  divided by ``factor``; sine and cosine times 0.1 ln(factor) + 1 (or ``gain``).
"""

from __future__ import annotations

import math

import torch

from . import kernels

_KEYS = {"linear": set(), "ntk": set(), "bands": {"context", "low", "high"}, "yarn": {"context", "fast", "slow", "gain"}}


def frequencies(rot: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """(radians per position of each of the rot / 2 pairs, fp64 on the host; the factor on sine and cosine)."""
    if rot < 0 or rot % 2 or not base > 0:
        raise ValueError(f"rotary: rot={rot}, base={base}")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-i / max(rot, 1)), 1.0
    s = dict(scaling)
    kind, factor = s.pop("kind", None), float(s.pop("factor", 0.0))
    if kind not in _KEYS or set(s) - _KEYS[kind] or not factor >= 1.0:
        raise ValueError(f"rotary: scaling {scaling}")
    if kind in ("bands", "yarn") and not float(s.get("context", 0)) > 0:
        raise ValueError(f"rotary: {kind} needs the trained context, got {scaling}")
    if kind == "ntk":
        if rot <= 2:
            raise ValueError("rotary: ntk needs more than one pair")
        return (base * factor ** (rot / (rot - 2))) ** (-i / rot), 1.0
    f = base ** (-i / max(rot, 1))
    if kind == "linear":
        return f / factor, 1.0
    if kind == "bands":
        low, high = float(s.get("low", 1.0)), float(s.get("high", 4.0))
        if not high > low:
            raise ValueError(f"rotary: bands need low < high, got {scaling}")
        kept = ((s["context"] * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f / factor * (1 - kept) + f * kept, 1.0
    pair = lambda turns: rot * math.log(s["context"] / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    first = max(math.floor(pair(float(s.get("fast", 32.0)))), 0)
    last = min(math.ceil(pair(float(s.get("slow", 1.0)))), rot - 1)
    stretched = ((i / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
    gain = s.get("gain")
    return f / factor * stretched + f * (1 - stretched), 0.1 * math.log(factor) + 1 if gain is None else float(gain)


class Rotary:
    """Norm and rotation of queries and keys: ``rotary(q, k, positions, norm=...)`` (``kernels.qk_norm_rope``)."""

    def __init__(self, head_dim: int, base: float = 10000.0, rot_dim: int | None = None, interleaved: bool = False,
                 scaling: dict | None = None, device=None):
        rot = head_dim if rot_dim is None else int(rot_dim)
        if head_dim <= 0 or head_dim % 8 or head_dim > 256 or rot % 16 or not 0 <= rot <= head_dim:
            raise ValueError(f"rotary: head size {head_dim} (a multiple of 8 up to 256), rot {rot} (of 16, up to it)")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        freq, self.gain = frequencies(rot, base, scaling)
        self.freq = freq.to(dev)
        self.head_dim, self.rot_dim, self.interleaved = head_dim, rot, bool(interleaved)

    def __call__(self, q: torch.Tensor, k: torch.Tensor, positions=None, norm: str | None = None, over: str = "head",
                 q_w=None, k_w=None, eps: float = 1e-6, out=None):
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"rotary: heads of {q.shape[-1]}, made for {self.head_dim}")
        return kernels.qk_norm_rope(q, k, self.freq, positions, gain=self.gain, interleaved=self.interleaved, norm=norm,
                                    over=over, q_w=q_w, k_w=k_w, eps=eps, out=out)
