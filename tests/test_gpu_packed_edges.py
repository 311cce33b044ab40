"""Packed attention where sequences, scores and probabilities reach their ends: no keys at all, against the formula."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _cu(c):
    return torch.tensor(c, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows", [[16], [40, 0, 300], [2000], [3] * 70])
def test_rows_without_any_keys_are_zero(gpu_lib, pkg, rows, causal, dtype):
    # no sequence has a key: every row sees none, whichever kernel the rows' number selects; the last row is of no sequence
    H, Hk, d, T = 8, 2, 64, sum(rows)
    q = torch.randn(T + 1, H, d, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    k = v = torch.empty(0, Hk, d, dtype=dtype, device=DEV)
    cq = [0]
    for n in rows:
        cq.append(cq[-1] + n)
    out = torch.full_like(q, 7.0)
    pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu([0] * len(cq)), causal=causal, out=out)
    assert bool((out[:T] == 0).all()) and bool((out[T:] == 7.0).all())
