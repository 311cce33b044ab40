"""Every form that the linears' launch plans choose among, with bias, activation, residual and alpha, gated and not, ragged in
every size, in both types, against 64 bits; the chosen form is asked for, so that a plan tuned anew cannot leave one out unseen."""

import ctypes

import pytest
import torch

from test_gpu_linear16 import ACTS, TYPES, _check, _check8, _inputs, _quantized

pytestmark = pytest.mark.gpu

# (1,000 x rows + weight rows of a workgroup, whether K is divided): (M, K, N) without and with a gate
FORMS16 = {
    (16, False): ((4, 600, 3336), None), (32, False): ((1, 7896, 6208), (3, 1584, 2512)), (64, False): ((13, 776, 13088), (14, 136, 12064)),
    (16064, False): ((69, 2544, 576), (350, 592, 496)), (48064, False): ((761, 920, 488), (196, 904, 1904)),
    (64128, False): ((1319, 56, 976), (241, 240, 1280)), (64128, True): ((269, 3856, 448), (565, 4960, 368)),
    (64256, False): ((482, 328, 6464), (921, 1032, 3456)), (64256, True): ((39, 4296, 15736), (1646, 2872, 544)),
    (128128, False): ((3499, 456, 1096), (578, 568, 6432)), (128128, True): ((1911, 4896, 368), (115, 6104, 6528)),
    (128256, False): ((2526, 464, 2680), (1077, 496, 5504)), (128256, True): ((548, 6096, 4120), (375, 5168, 4944)),
    (192256, False): ((1389, 600, 6160), (1198, 1784, 7216)), (192256, True): ((3226, 7688, 1120), (1826, 6880, 1408)),
    (256256, False): ((2918, 584, 9576), (933, 456, 14000)), (256256, True): ((4081, 7944, 1040), (1687, 6800, 2656)),
}
FORMS8 = {
    (16, False): ((2, 992, 992), None), (32, False): ((9, 1040, 5576), (14, 880, 1088)), (64, False): ((13, 544, 13864), (10, 176, 14912)),
    (16064, False): ((52, 2544, 264), (24, 336, 4736)), (32064, False): ((39, 3728, 5528), (25, 944, 9472)),
    (48064, False): ((206, 688, 2456), (42, 736, 11328)), (64064, False): ((259, 1696, 5856), (62, 1504, 8320)),
    (128064, False): ((581, 592, 2496), (70, 928, 13568)), (64256, False): ((1205, 1568, 3312), (2062, 592, 1536)),
    (64256, True): ((168, 7632, 10432), (1282, 7088, 1536)), (128256, False): ((2169, 752, 2080), (3851, 432, 1920)),
    (128256, True): ((1763, 6896, 1664), (2330, 8176, 896)), (192256, False): ((521, 2272, 14328), (1918, 752, 11776)),
    (192256, True): ((4543, 6448, 832), (865, 6736, 4672)), (256256, False): ((4088, 288, 6248), (2218, 272, 12224)),
}


def _cases(forms):
    return [pytest.param(form, shape, gated, id=f"{form[0]}{'-divided' if form[1] else ''}{'-gated' if gated else ''}-{'x'.join(map(str, shape))}")
            for form, shapes in forms.items() for gated, shape in enumerate(shapes) if shape]


def _form(query, M, K, N, gated):
    splits = ctypes.c_int()
    return query(M, K, N, int(gated), ctypes.byref(splits)), splits.value > 1


@pytest.mark.parametrize("form,shape,gated", _cases(FORMS16))
@pytest.mark.parametrize("dtype", TYPES)
def test_16_bits(gpu_lib, pkg, form, shape, gated, dtype):
    M, K, N = shape
    assert _form(gpu_lib.linear16_tile, M, K, N, gated) == form
    x, w, b, r = _inputs(M, K, N, dtype, bool(gated), seed=K)
    lin = pkg.linear.Linear16.from_float(w, b, gated=bool(gated), dtype=dtype)
    assert torch.equal(lin.weight, w.to(dtype))
    for act, res, alpha in ((ACTS[K // 8 % 4 + 1], r, -0.5), (None, None, 1.0)):
        _check(lin(x, act, res, alpha), x, lin.weight, lin.bias, act, bool(gated), res, alpha)


@pytest.mark.parametrize("form,shape,gated", _cases(FORMS8))
@pytest.mark.parametrize("dtype", TYPES)
def test_e4m3(gpu_lib, pkg, form, shape, gated, dtype):
    M, K, N = shape
    assert _form(gpu_lib.f8_linear_tile, M, K, N, gated) == form
    x, w, b, r = _inputs(M, K, N, dtype, bool(gated), seed=K)
    lin = pkg.f8.F8Linear.from_float(w, bias=b, gated=bool(gated))
    act = ACTS[K // 16 % 4 + 1]
    _check8(lin(x, act, r, -0.5), _quantized(x), lin, b, act, r, -0.5, dtype)
    _, rows = pkg.norm.AddNorm(torch.ones(K))(x, f8=True)
    _check8(lin(rows, act, r, -0.5), rows.dequantized().double(), lin, b, act, r, -0.5, dtype)
