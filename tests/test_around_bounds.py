"""CPU tests of the bounds that the GPU tests hold the linears' end to."""

import numpy as np
import pytest
import torch

from oracle import around as A

F = np.float32


def _fma(a, b, c):
    return (a.astype(np.float64) * np.asarray(b, np.float64) + np.asarray(c, np.float64)).astype(F)


def _gelu(z, reciprocal, power):
    """The kernel's steps in fp32, its reciprocal and power of two off by so many steps."""
    off = lambda v, steps: (v * (1 + steps * 2.0 ** -23)).astype(F)  # noqa: E731
    t = off(1 / _fma(np.abs(z), F(F(0.3275911) * F(0.70710678)), F(1)).astype(np.float64), reciprocal)
    q = _fma(t, F(1.061405429), F(-1.453152027))
    for c in (1.421413741, -0.284496736, 0.254829592):
        q = _fma(t, q, F(c))
    tail = F(0.5) * t * q * off(np.exp2((F(-0.72134752) * z * z).astype(np.float64)), power)
    return np.where(z > 0, F(1) - tail, tail), (z * np.where(z > 0, F(1) - tail, tail)).astype(F)


@pytest.mark.parametrize("reciprocal", [-1, 0, 1])
@pytest.mark.parametrize("power", [-1, 0, 1])
def test_gelu_in_fp32_keeps_its_bound(reciprocal, power):
    z = np.concatenate([np.linspace(-13, 13, 400001), np.linspace(-0.3, 0.3, 200001)]).astype(F)
    p, y = _gelu(z, reciprocal, power)
    ref, bound = A.activate(torch.from_numpy(z).double(), "gelu")
    assert bool(((torch.from_numpy(y).double() - ref).abs() <= bound + 2.0 ** -126).all())
    off = np.abs(p - torch.special.ndtr(torch.from_numpy(z).double()).numpy())
    assert off.max() <= 5.6e-7 and off[z < -1].max() <= 1.8e-7
