"""Edges of the residual's norm, the linears with an end and the cache in 4 bits that their first tests do not reach."""

import pytest
import torch

from test_gpu_linear16 import _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("K", [8, 64, 136, 192, 328])  # an odd count of 64s: the last block of 128 k holds one
@pytest.mark.parametrize("M,N", [(1, 128), (16, 200), (5, 5000), (9, 10240)])  # 16, 16, 32 and 64 weight rows a workgroup
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_behind_a_piece_reach_nothing(gpu_lib, pkg, K, M, N, dtype):
    """What lies behind a piece of 64 weight rows, another piece or other memory, takes no part in its outputs."""
    x, w, _, _ = _inputs(M, K, N, dtype)
    lin = pkg.linear.Linear16.from_float(w, dtype=dtype)
    want = lin(x)
    assert bool(torch.isfinite(want).all())
    # other memory behind the last: the packed weights at the head of a buffer of NaN
    n = lin.packed.numel()
    behind = torch.full((n + 65536,), 255, dtype=torch.uint8, device=DEV)
    behind[:n] = lin.packed
    assert torch.equal(pkg.kernels.linear16(x, behind[:n], N), want)
    # other pieces: infinite and NaN weights in every second
    rows = torch.arange(N, device=DEV) // 64 % 2 == 1
    w[rows, 0], w[rows, K - 1] = float("inf"), float("nan")
    y = pkg.linear.Linear16.from_float(w, dtype=dtype)(x)
    assert torch.equal(y[:, ~rows], want[:, ~rows]) and bool(y[:, rows].isnan().all())
