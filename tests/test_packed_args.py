"""CPU tests of the packed-row operators: argument checks of the C ABI before any launch, and the rotary frequencies."""

import ctypes
import math

import pytest
import torch

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 4)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.capi.lib(require_gpu=False)


def _rope(lib, T=4, H=4, Hk=2, d=64, rot=64, norm=1, row=0, dtype=0, eps=1e-6, st=512, sh=64, q=P, freq=P, w=None):
    return lib.qk_norm_rope(q, P, P, P, st, sh, st, sh, st, sh, st, sh, w, 0, None, 0, eps, None, 0, freq, 1.0, T, H,
                            Hk, d, rot, norm, row, 0, dtype, None)


def test_qk_norm_rope_refusals(lib):
    assert _rope(lib, T=0) == 0
    for kw in (dict(T=-1), dict(H=0), dict(Hk=0), dict(d=0), dict(rot=80), dict(eps=-1.0), dict(eps=math.nan),
               dict(T=1 << 22)):
        assert _rope(lib, **kw) == -2, kw
    for kw in (dict(d=60, rot=48), dict(d=264), dict(rot=24), dict(norm=3), dict(dtype=2), dict(H=1030, row=1)):
        assert _rope(lib, **kw) == -4, kw
    for kw in (dict(st=60), dict(st=32), dict(sh=4), dict(sh=-64), dict(st=1 << 24), dict(q=ODD), dict(w=ODD),
               dict(freq=ODD)):
        assert _rope(lib, **kw) == -3, kw
    assert _rope(lib, q=None) == -1 and _rope(lib, freq=None) == -1


def _attn(lib, n=2, Tq=8, Tk=8, H=4, Hk=2, d=64, scale=0.125, dtype=0, st=256, sh=64, q=P, cu=P, ws=None, nbytes=0):
    return lib.packed_attention(q, P, P, P, st, sh, st, sh, st, sh, st, sh, cu, P, n, Tq, Tk, H, Hk, d, 0, scale, dtype,
                                ws, nbytes, None)


def test_packed_attention_refusals(lib):
    assert _attn(lib, n=0) == 0 and _attn(lib, Tq=0) == 0
    for kw in (dict(n=-1), dict(Tq=-1), dict(Tk=-1), dict(H=0), dict(H=5), dict(d=0), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(Tq=1 << 30, st=256)):
        assert _attn(lib, **kw) == -2, kw
    for kw in (dict(d=60), dict(d=136), dict(dtype=3)):
        assert _attn(lib, **kw) == -4, kw
    for kw in (dict(st=36), dict(st=32), dict(sh=12), dict(st=1 << 24), dict(q=ODD), dict(cu=ctypes.c_void_p(4098))):
        assert _attn(lib, **kw) == -3, kw
    assert _attn(lib, q=None) == -1 and _attn(lib, cu=None) == -1
    # few rows against many keys: partials in a workspace of a stated size
    need = lib.packed_attention_workspace_bytes(2, 2, 10000, 4, 2, 64)
    assert need > 0
    assert _attn(lib, Tq=2, Tk=10000) == -2 and _attn(lib, Tq=2, Tk=10000, ws=P, nbytes=need - 1) == -2
    assert _attn(lib, Tq=2, Tk=10000, ws=ctypes.c_void_p((1 << 20) + 16), nbytes=need) == -3
    assert lib.packed_attention_workspace_bytes(1, 8192, 8192, 32, 8, 128) == 0
    assert lib.packed_attention_workspace_bytes(0, 0, 0, 4, 2, 64) == 0


def test_rotary_frequencies(pkg):
    fr = pkg.rotary.frequencies
    f, gain = fr(64)
    assert f.dtype == torch.float64 and gain == 1.0 and f[0] == 1.0
    assert float((f - 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).abs().max()) == 0
    assert torch.equal(fr(64, scaling={"kind": "linear", "factor": 4.0})[0], f / 4)
    g, _ = fr(64, scaling={"kind": "ntk", "factor": 4.0})
    assert g[0] == f[0] and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12  # the slowest pair stretched by the factor
    for kind in ("bands", "yarn"):
        b, gain = fr(128, 500000.0, {"kind": kind, "factor": 8.0, "context": 8192})
        a, _ = fr(128, 500000.0)
        assert b[0] == a[0] and abs(float(b[-1] / a[-1]) - 0.125) < 1e-12 and bool((b[1:] < b[:-1]).all())
        assert gain == (1.0 if kind == "bands" else 0.1 * math.log(8.0) + 1)
    assert fr(64, scaling={"kind": "yarn", "factor": 2.0, "context": 512, "gain": 1.5})[1] == 1.5
    assert fr(0)[0].numel() == 0
    for bad in (dict(rot=63), dict(rot=64, base=0.0), dict(rot=64, scaling={"kind": "other", "factor": 2.0}),
                dict(rot=64, scaling={"kind": "linear"}), dict(rot=64, scaling={"kind": "yarn", "factor": 2.0}),
                dict(rot=64, scaling={"kind": "linear", "factor": 2.0, "context": 9}),
                dict(rot=64, scaling={"kind": "bands", "factor": 2.0, "context": 9, "low": 4.0, "high": 1.0}),
                dict(rot=2, scaling={"kind": "ntk", "factor": 2.0})):
        with pytest.raises(ValueError):
            fr(**bad)
    for bad in (dict(head_dim=60), dict(head_dim=264), dict(head_dim=64, rot_dim=24), dict(head_dim=64, rot_dim=80)):
        with pytest.raises(ValueError):
            pkg.rotary.Rotary(device="cpu", **bad)


def test_f8_refusals(lib):
    def linear(M=4, K=256, N=128, st=256, dtype=0, x=P, y=P, ws=None, n=0):
        return lib.f8_linear(x, st, P, P, y, M, K, N, dtype, ws, n, None)

    assert linear(M=0) == 0
    for kw in (dict(M=-1), dict(K=0), dict(K=250), dict(N=0), dict(N=100), dict(K=1 << 21, st=1 << 21),
               dict(M=1 << 23, N=1 << 20)):
        assert linear(**kw) == -2, kw
    assert linear(dtype=2) == -4
    for kw in (dict(st=260), dict(st=128), dict(x=ODD), dict(y=ODD)):
        assert linear(**kw) == -3, kw
    assert linear(x=None) == -1 and linear(y=None) == -1
    need = lib.f8_linear_workspace_bytes(238, 5120, 2560)
    assert need > 238 * 5120 and lib.f8_linear_workspace_bytes(16, 5120, 2560) == 0
    assert linear(M=238, K=5120, N=2560, st=5120, ws=P, n=need - 1) == -2
    assert linear(M=238, K=5120, N=2560, st=5120, ws=ctypes.c_void_p((1 << 20) + 16), n=need) == -3
    splits = ctypes.c_int(7)
    assert lib.f8_linear_partials(P, 256, P, P, P, 16, ctypes.byref(splits), 4, 256, 128, 0, None, 0, None) == -2
    assert splits.value == 0
    assert lib.f8_linear_partials(P, 256, P, P, P, 1 << 20, None, 4, 256, 128, 0, None, 0, None) == -1
    assert lib.f8_packed_codes_bytes(65, 129) == 0 and lib.f8_packed_codes_bytes(72, 144) == 2 * 2 * 8192
    assert lib.f8_pack_codes(None, P, 64, 128, None) == -1 and lib.f8_pack_codes(P, P, 64, 100, None) == -2
    assert lib.f8_quantize_weight(None, P, P, 64, 128, None) == -1


def test_short_way_takes_the_ordinary_case_only(pkg, lib):
    # the native module answers None for whatever it does not take, and the wrappers then refuse with their messages
    b = pkg.capi.bind
    assert pkg.build.library_hash(pkg.build.BIND_PATH) == pkg.build.source_hash()
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    assert b.packed_attention(x, x, x, cu, None, False, None, 0, 0) is None          # host tensors
    assert b.packed_attention(x) is None and b.packed_attention(1, 2, 3, 4, 5, 6, 7, 8, 9) is None
    assert b.qk_norm_rope(x, x, cu, None, 1.0, False, 0, False, None, None, 1e-6) is None
    assert b.f8_linear(x[:, 0], cu, cu, 64, 0, 0) is None and b.f8_linear("x", cu, cu, 64, 0, 0) is None
    with pytest.raises(TypeError):
        b.connect(1, 2)
    assert set(pkg.capi._SHORT) <= set(pkg.capi.SIGNATURES)
