"""CPU tests of the residual's norm, the linears' end and the cache in 4 bits: argument checks of the C ABI before any launch,
workspaces and layouts over sizes of every kind, and the 64-bit restatements themselves."""

import ctypes
import math
import random

import pytest
import torch

from oracle import cache4 as C4

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 4)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.capi.lib(require_gpu=False)


def _norm(lib, x=P, y=P, s=P, h=P, hq=None, hs=None, w=None, eps=1e-6, norm=1, alpha=1.0, st=64, s_st=64, T=4, D=64, dtype=0, fp32=0):
    return lib.add_norm(x, fp32, y, alpha, s, h, hq, hs, w, None, eps, norm, st, st, s_st, 64, T, D, dtype, None)


def test_add_norm_refusals(lib):
    assert _norm(lib, T=0) == 0
    for kw in (dict(T=-1), dict(D=0), dict(D=60), dict(D=32776), dict(T=(1 << 24) + 1), dict(eps=-1.0), dict(eps=math.nan), dict(alpha=math.inf),
               dict(h=None, hq=P, hs=P, D=72)):
        assert _norm(lib, **kw) == -2, kw
    for kw in (dict(norm=0), dict(norm=3), dict(dtype=2)):
        assert _norm(lib, **kw) == -4, kw
    for kw in (dict(st=60), dict(s_st=32), dict(s_st=0), dict(x=ODD), dict(w=ODD), dict(h=ODD), dict(s=ODD)):
        assert _norm(lib, **kw) == -3, kw
    for kw in (dict(x=None), dict(h=None), dict(hq=P, hs=P), dict(h=None, hq=P)):
        assert _norm(lib, **kw) == -1, kw


def _linear16(lib, x=P, wp=P, bias=None, r=None, r_st=64, alpha=1.0, act=0, gated=0, y=P, M=4, K=64, N=64, x_st=64, dtype=0, ws=None, n=0):
    return lib.linear16(x, x_st, wp, bias, r, r_st, alpha, act, gated, y, M, K, N, dtype, ws, n, None)


def test_linear16_refusals(lib):
    assert _linear16(lib, M=0) == 0
    for kw in (dict(M=-1), dict(K=0), dict(K=60), dict(N=0), dict(N=60), dict(N=24, gated=1), dict(K=(1 << 20) + 8), dict(M=(1 << 24) + 1),
               dict(M=1 << 23, N=1 << 20), dict(alpha=math.nan)):
        assert _linear16(lib, **kw) == -2, kw
    for kw in (dict(dtype=2), dict(act=-1), dict(act=5)):
        assert _linear16(lib, **kw) == -4, kw
    for kw in (dict(x_st=60), dict(x_st=56), dict(x_st=(1 << 21) + 8), dict(r=P, r_st=56), dict(r=P, r_st=68), dict(x=ODD), dict(y=ODD), dict(bias=ODD),
               dict(r=ODD), dict(wp=ODD)):
        assert _linear16(lib, **kw) == -3, kw
    assert _linear16(lib, x=None) == -1 and _linear16(lib, wp=None) == -1 and _linear16(lib, y=None) == -1
    need = lib.linear16_workspace_bytes(1000, 10240, 2560, 0)
    assert need > 0
    big = dict(M=1000, K=10240, N=2560, x_st=10240)
    assert _linear16(lib, **big) == -2 and _linear16(lib, **big, ws=P, n=need - 1) == -2
    assert _linear16(lib, **big, ws=ctypes.c_void_p((1 << 20) + 16), n=need) == -3
    assert lib.linear16_packed_bytes(72, 72, 0) == 2 * 2 * 8192 and lib.linear16_packed_bytes(72, 72, 1) == 0 and lib.linear16_packed_bytes(80, 72, 1) == 2 * 2 * 8192
    assert lib.linear16_pack(None, P, 64, 64, 0, None) == -1 and lib.linear16_pack(P, P, 64, 60, 0, None) == -2 and lib.linear16_pack(ODD, P, 64, 64, 0, None) == -3


def test_f8_linear_end_refusals(lib):
    def call(x=P, x_st=256, xq=None, sx=None, qp=P, bias=None, r=None, act=0, gated=0, y=P, M=4, K=256, N=128, dtype=0, ws=None, n=0):
        return lib.f8_linear_end(x, x_st, xq, sx, qp, P, bias, r, 128, 1.0, act, gated, y, M, K, N, dtype, ws, n, None)

    assert call(M=0) == 0
    for kw in (dict(M=-1), dict(K=250), dict(N=100), dict(N=96, gated=1), dict(K=1 << 21), dict(M=1 << 23, N=1 << 20), dict(M=(1 << 24) - 1, K=1 << 20)):
        assert call(**kw) == -2, kw
    assert call(dtype=2) == -4 and call(act=7) == -4
    for kw in (dict(x_st=260), dict(x_st=128), dict(x=ODD), dict(y=ODD), dict(bias=ODD)):
        assert call(**kw) == -3, kw
    for kw in (dict(x=None), dict(xq=P, sx=P), dict(x=None, xq=P), dict(qp=None), dict(y=None)):
        assert call(**kw) == -1, kw
    need = lib.f8_linear_end_workspace_bytes(238, 5120, 2560, 0, 0)
    assert need > 238 * 5120 and lib.f8_linear_end_workspace_bytes(16, 5120, 2560, 0, 0) == 0
    assert lib.f8_linear_end_workspace_bytes(238, 5120, 2560, 0, 1) < 238 * 5120
    assert call(M=238, K=5120, N=2560, x_st=5120, ws=P, n=need - 1) == -2
    assert call(M=238, K=5120, N=2560, x_st=5120, ws=ctypes.c_void_p((1 << 20) + 16), n=need) == -3
    assert lib.f8_rows_bytes(17, 130) == 32 * 256 and lib.f8_rows_scales_bytes(17, 130) == 32 * 2 * 4 + 1024 and lib.f8_rows_bytes(0, 130) == 0


def _attend(lib, q=P, o=P, st=512, sh=64, data=P, cu=P, table=P, n=2, T=4, H=8, Hk=2, d=64, pages=3, width=2, scale=0.1, dtype=1, ws=None, nbytes=0):
    return lib.cache4_attention(q, o, st, sh, st, sh, data, cu, P, table, n, T, H, Hk, d, pages, width, 1, scale, dtype, ws, nbytes, None)


def test_cache4_refusals(lib):
    assert _attend(lib, n=0) == 0 and _attend(lib, T=0) == 0
    for kw in (dict(n=-1), dict(T=-1), dict(H=0), dict(Hk=0), dict(H=7), dict(d=0), dict(pages=-1), dict(width=-1), dict(scale=0.0), dict(scale=math.nan),
               dict(scale=math.inf), dict(T=1 << 24), dict(width=1 << 23), dict(T=(1 << 23) - 1, H=1 << 10, Hk=1)):
        assert _attend(lib, **kw) == -2, kw
    for kw in (dict(d=60), dict(d=136), dict(dtype=2)):
        assert _attend(lib, **kw) == -4, kw
    for kw in (dict(st=516), dict(st=32), dict(sh=12), dict(q=ODD), dict(data=ODD), dict(cu=ctypes.c_void_p(4098)), dict(table=ctypes.c_void_p(4098))):
        assert _attend(lib, **kw) == -3, kw
    for kw in (dict(q=None), dict(o=None), dict(cu=None), dict(table=None), dict(data=None)):
        assert _attend(lib, **kw) == -1, kw
    need = lib.cache4_attention_workspace_bytes(2, 4, 100, 8, 2, 64)
    assert need > 0 and _attend(lib, width=100) == -2 and _attend(lib, width=100, ws=P, nbytes=need - 1) == -2
    assert _attend(lib, width=100, ws=ctypes.c_void_p((1 << 20) + 16), nbytes=need) == -3
    append = lambda k=P, st=128, T=4, dtype=1, **kw: lib.cache4_append(k, P, st, 64, 128, 64, P, P, P, P, 2, T, 2, 64, 3, 2, dtype, None)  # noqa: E731
    assert append(T=0) == 0 and append(k=None) == -1 and append(st=100) == -3 and append(k=ODD) == -3 and append(dtype=5) == -4 and append(T=-1) == -2
    read = lambda k=P, T=4, d=64: lib.cache4_read(k, P, P, P, P, P, 2, T, 2, d, 3, 2, 1, None)  # noqa: E731
    assert read(T=0) == 0 and read(k=None) == -1 and read(k=ODD) == -3 and read(d=60) == -4
    assert lib.cache4_bytes(3, 2, 64) == 3 * 2 * 64 * 72 and lib.cache4_bytes(3, 2, 80) == 3 * 2 * 64 * 144 and lib.cache4_bytes(0, 2, 64) == 0
    assert lib.cache4_bytes(1, 2, 136) == 0


def test_workspaces_over_sizes(lib):
    rng = random.Random(0)
    for _ in range(400):
        M, K, N = (int(math.exp(rng.uniform(0, 9))) for _ in range(3))
        K, N = 16 * K, 64 * N
        for gated in (0, 1):
            assert lib.linear16_workspace_bytes(M, K, N, gated) >= 0 and lib.linear16_packed_bytes(N, K, gated) >= 2 * N * K
            assert lib.f8_linear_end_workspace_bytes(M, K, N, gated, 0) >= lib.f8_linear_end_workspace_bytes(M, K, N, gated, 1)
        n, T, width = rng.randrange(1, 200), rng.randrange(1, 3000), int(math.exp(rng.uniform(0, 9))) - 1
        assert (lib.cache4_attention_workspace_bytes(n, T, width, 8, 2, 128) > 0) <= (width > 8)


def test_the_cache_restated(pkg):
    x = torch.randn(50, 3, 80, generator=torch.Generator().manual_seed(0)).bfloat16()
    x[3], x[4], x[5] = 0, 7.0, x[5] * 1e-30
    c, s, z = C4.hold(x)
    assert float((s * (c - z) - x.double()).abs().max()) <= float(0.5 * s.max() + 1e-9)
    assert bool((s * (c - z) == 0)[3].all()) and torch.equal(s, s.float().bfloat16().double())
    q = torch.randn(2, 6, 80).bfloat16()
    o, bound = C4.attention(q, (c, s, z), (c, s, z), True, 0.1)
    plain = (s * (c - z))[:49]  # what the first row sees
    p = torch.softmax(0.1 * torch.einsum("hd,khd->hk", q[0].double(), plain.repeat_interleave(2, 1)), 1)
    assert torch.allclose(o[0], torch.einsum("hk,khd->hd", p, plain.repeat_interleave(2, 1))) and bool((bound > 0).all())
    assert pkg.cache4.PAGE == 64


def test_gated_rows_are_a_permutation(pkg):
    for N in (64, 128, 640):
        order = pkg.f8._gated_rows(N, "cpu")
        assert sorted(order.tolist()) == list(range(N))
        # rows 16 g + 4 j + e of piece p: even j gates, odd j up values, of output 32 p + 8 g + 4 (j / 2) + e
        for r in (0, 5, 17, 63):
            g, j, e = r // 16, r % 16 // 4, r % 4
            assert int(order[r]) == 8 * g + 4 * (j // 2) + e + (N // 2) * (j % 2)


def test_the_norm_and_the_activations_restated(pkg):
    import torch.nn.functional as F

    from oracle import around as A
    g = torch.Generator().manual_seed(1)
    x, y, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).float() for s in ((5, 40), (5, 40), (40,), (40,)))
    s, _, h, bound = A.add_norm(x, y, 0.5, w, b, "layer", 1e-5)
    assert torch.allclose(h, F.layer_norm(x.double() + 0.5 * y.double(), (40,), w.double(), b.double(), 1e-5), rtol=1e-12, atol=1e-12)
    _, _, h, _ = A.add_norm(x, None, 1.0, w, None, "rms", 1e-6)
    assert torch.allclose(h, F.rms_norm(x.double(), (40,), w.double(), 1e-6), rtol=1e-12, atol=1e-12) and bool((bound > 0).all())
    z = torch.cat([torch.linspace(-30, 30, 601, dtype=torch.float64), torch.tensor([0.0, -0.0, 1e-30])])
    for kind, ref in ((None, lambda t: t), ("relu", F.relu), ("gelu", F.gelu), ("gelu_tanh", lambda t: F.gelu(t, approximate="tanh")), ("silu", F.silu)):
        assert torch.allclose(A.activate(z, kind)[0], ref(z), rtol=1e-9, atol=1e-12), kind
    z, res = torch.randn(3, 8, generator=g, dtype=torch.float64), torch.randn(3, 4, generator=g).half()
    y, _ = A.end(z, torch.zeros_like(z), w[:8], "silu", True, res, 2.0, torch.float16)
    u = z + w[:8].double()
    assert torch.allclose(y, res.double() + 2 * F.silu(u[:, :4]) * u[:, 4:], rtol=1e-9, atol=1e-12)


def test_the_step_is_the_least_that_reaches(pkg):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(200, 1, 64, generator=g) * torch.exp(4 * torch.randn(200, 1, 1, generator=g)) + 3 * torch.randn(200, 1, 1, generator=g)
    x = x.bfloat16().double()
    _, s, _ = C4.hold(x)
    s = s[..., :1]
    less = (s.float().view(torch.int32) - (1 << 16)).view(torch.float32).double()  # the bf16 value below
    lo, hi, far = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True), x.abs().amax(-1, keepdim=True)
    reaches = lambda t: (15 * t >= hi - lo) & (120 * t >= far)  # noqa: E731
    assert bool(reaches(s).all()) and not bool(reaches(less).any())
