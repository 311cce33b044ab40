"""Layouts of the e4m3 linear's input that it cannot read where they lie: copied first, the same bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [2, 16, 40, 238])
def test_layouts_that_are_copied(gpu_lib, pkg, M, dtype):
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, 256, generator=g, device=DEV).to(dtype)
    lin = pkg.f8.F8Linear.from_float(torch.randn(192, 256, generator=g, device=DEV))
    ref = lin(x)
    columns = x.t().contiguous().t()                       # a row's values M apart
    assert columns.stride(1) != 1 and torch.equal(lin(columns), ref)
    wide = torch.zeros(M, 260, dtype=dtype, device=DEV)    # rows 260 apart: aligned at the first, at no other
    wide[:, :256] = x
    assert wide.stride(0) % 8 and torch.equal(lin(wide[:, :256]), ref)
    same = x[:1].expand(M, 256)                            # one row M times
    assert same.stride(0) == 0 and torch.equal(lin(same), lin(same.contiguous()))
    lapped = x.reshape(-1)[:(M - 1) * 64 + 256].as_strided((M, 256), (64, 1))  # rows that share values
    assert torch.equal(lin(lapped), lin(lapped.contiguous()))
    deep = x.view(M, 2, 128).transpose(0, 1).contiguous().transpose(0, 1)       # [M, 2, 128] of another order
    assert torch.equal(lin(deep.reshape(M, 256)), ref)
    parts, n = lin.partials(columns)
    acc = parts[0].clone()
    for s in range(1, n):
        acc += parts[s]
    assert torch.equal(acc.to(dtype), ref)
