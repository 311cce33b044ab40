"""The residual's addition and the norm in one pass, in 16 bits and in e4m3, against 64 bits."""

import pytest
import torch

from oracle import around as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _inputs(T, D, stream, dtype, seed=0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x = r(T, D) * (1 + 9 * (torch.rand(D, generator=g, device=DEV) < 0.05)) + shift
    return x.to(stream), (0.5 * r(T, D)).to(dtype), 1 + 0.2 * r(D), 0.3 * r(D)


def _within(got, ref, bound):
    worst = float(((got.double() - ref).abs() / bound).max()) if ref.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.2f} of its bound"


def _check(s, h, x, y, alpha, w, b, norm, eps):
    rs, bs, rh, bh = O.add_norm(x, y, alpha, w, b, norm, eps)
    _within(s, rs, bs)
    _within(h, rh, bh + O.HALF_STEP[h.dtype] * (rh.abs() + bh) + O.SMALLEST[h.dtype])


def _check8(rows, x, y, alpha, w, b, norm, eps):
    _, _, rh, bh = O.add_norm(x, y, alpha, w, b, norm, eps)
    T, D = rh.shape
    kb = -(-D // 128)
    pad = lambda t: torch.nn.functional.pad(t, (0, kb * 128 - D)).view(T, kb, 128)  # noqa: E731
    top, slack = pad(rh.abs()).amax(-1), pad(bh).amax(-1)
    scale = top.clamp_min(O.FLOOR) / O.TOP
    _within(rows.scales, scale, (slack + 4 * 2.0 ** -24 * top) / O.TOP + 2.0 ** -140)
    # a code: half a step of e4m3 (2^-4 of the value, 2^-10 of the scale among the smallest) off the value the kernel had
    each = scale.repeat_interleave(128, 1)[:, :D]
    _within(rows.dequantized(), rh, (2.0 ** -4 + 2.0 ** -20) * (rh.abs() + bh) + 2 * bh + (2.0 ** -10 + 2.0 ** -20) * each)


@pytest.mark.parametrize("D", [8, 24, 640, 1104, 2560, 4096, 4104, 5120, 8192, 20000, 32768])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_against_the_definition(gpu_lib, pkg, D, dtype, norm):
    for T, stream in ((1, dtype), (3, torch.float32), (17, dtype), (1500 if D <= 5120 else 33, torch.float32)):
        x, y, w, b = _inputs(T, D, stream, dtype, seed=D + T)
        s, h = pkg.kernels.add_norm(x, y, w, b if norm == "layer" else None, norm=norm, eps=1e-5)
        assert s.dtype is stream and h.dtype is dtype
        _check(s, h, x, y, 1.0, w, b if norm == "layer" else None, norm, 1e-5)


@pytest.mark.parametrize("D", [16, 112, 128, 656, 2560, 5120, 8208, 32768])
@pytest.mark.parametrize("dtype", TYPES)
def test_in_e4m3(gpu_lib, pkg, D, dtype):
    for T, norm, stream in ((1, "rms", dtype), (16, "layer", torch.float32), (17, "rms", torch.float32), (1100, "layer", dtype)):
        if T * D > 6e6:
            T = 40
        x, y, w, b = _inputs(T, D, stream, dtype, seed=D + T)
        s, rows = pkg.norm.AddNorm(w, b, norm=norm, eps=1e-6)(x, y, 0.75, f8=True)
        _check8(rows, x, y, 0.75, w, b, norm, 1e-6)
        rs, bs, _, _ = O.add_norm(x, y, 0.75, w, b, norm, 1e-6)
        _within(s, rs, bs)
        assert rows.shape == (T,) and rows.features == D and rows.dtype is dtype


@pytest.mark.parametrize("f8", [False, True])
def test_strides_in_place_and_what_lies_beside(gpu_lib, pkg, f8):
    for T in (5, 1030):
        wide = _inputs(T, 3 * 640, torch.float16, torch.float16, seed=T)[0]
        keep = wide.clone()
        x, y = wide[:, 640:1280], wide[:, 1280:]
        x0, y0 = x.clone(), y.clone()
        w = torch.rand(640, device=DEV) + 0.5
        if f8:
            s, packed = pkg.kernels.add_norm_f8(x, y, w, alpha=-2.0, sum_out=x)
            h = None
        else:
            buf = torch.full((T, 1280), 7.0, dtype=torch.float16, device=DEV)
            s, h = pkg.kernels.add_norm(x, y, w, alpha=-2.0, sum_out=x, out=buf[:, 320:960])
            assert bool((buf[:, :320] == 7).all() and (buf[:, 960:] == 7).all())
        assert s.data_ptr() == x.data_ptr()
        assert torch.equal(wide[:, :640], keep[:, :640]) and torch.equal(wide[:, 1280:], keep[:, 1280:])
        if f8:
            _check8(pkg.f8.F8Rows(*packed, (T,), 640, torch.float16), x0, y0, -2.0, w, None, "rms", 1e-6)
            rs, bs, _, _ = O.add_norm(x0, y0, -2.0, w, None, "rms", 1e-6)
            _within(s, rs, bs)
        else:
            _check(s, h, x0, y0, -2.0, w, None, "rms", 1e-6)


def test_without_a_branch(gpu_lib, pkg):
    x, _, w, b = _inputs(40, 2560, torch.float32, torch.bfloat16)
    s, h = pkg.kernels.add_norm(x, None, w, b, norm="layer", dtype=torch.bfloat16)
    assert s is x
    _check(s, h, x, None, 1.0, w, b, "layer", 1e-6)
    s, h = pkg.kernels.add_norm(x.half())
    _check(s, h, x.half(), None, 1.0, None, None, "rms", 1e-6)


def test_a_mean_far_from_zero(gpu_lib, pkg):
    x, y, w, b = _inputs(9, 5120, torch.float32, torch.float16, shift=300.0)
    s, h = pkg.kernels.add_norm(x, y, w, b, norm="layer", eps=0.0)
    _check(s, h, x, y, 1.0, w, b, "layer", 0.0)


def test_zeros_infinities_and_nan(gpu_lib, pkg):
    x, y, w, _ = _inputs(6, 640, torch.float32, torch.float16)
    x[0], y[0] = 0.0, 0.0
    x[2, 5], x[4, 600] = float("nan"), float("inf")
    s, h = pkg.kernels.add_norm(x, y, w)
    assert bool((h[0] == 0).all()) and bool(h[2].isnan().all())
    assert bool(torch.isfinite(h[[1, 3, 5]]).all()) and bool((h[4].isnan() | (h[4] == 0)).all()) and bool(h[4, 600].isnan())
    _, packed = pkg.kernels.add_norm_f8(x, y, w)
    rows = pkg.f8.F8Rows(*packed, (6,), 640, torch.float16)
    d = rows.dequantized()
    assert bool((d[0] == 0).all()) and bool(d[2].isnan().all()) and bool(torch.isfinite(d[[1, 3, 5]]).all())
    assert bool(d[4, 512:].isnan().all())  # the block of the infinity


def test_no_rows_and_leading_dimensions(gpu_lib, pkg):
    n = pkg.norm.AddNorm(torch.ones(64), norm="layer")
    s, h = n(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV, dtype=torch.float16))
    assert s.shape == h.shape == (0, 64) and h.dtype is torch.float16
    s, rows = n(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV, dtype=torch.float16), f8=True)
    assert rows.rows == 0 and rows.dequantized().shape == (0, 64)
    x, y, _, _ = _inputs(24, 64, torch.float32, torch.float16)
    s, h = n(x.view(2, 3, 4, 64), y.view(2, 3, 4, 64), out=torch.empty(2, 3, 4, 64, device=DEV, dtype=torch.float16))
    s2, h2 = n(x, y)
    assert torch.equal(s.view(24, 64), s2) and torch.equal(h.view(24, 64), h2)
    s, rows = n(x.view(2, 12, 64), y.view(2, 12, 64), f8=True)
    assert rows.shape == (2, 12) and rows.dequantized().shape == (2, 12, 64)


@pytest.mark.parametrize("T", [4, 1200])
def test_captured_and_replayed(gpu_lib, pkg, T):
    x, y, w, _ = _inputs(T, 2560, torch.float32, torch.float16)
    n = pkg.norm.AddNorm(w)
    n(x, y), n(x, y, f8=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, h = n(x, y)
        _, rows = n(x, y, f8=True)
    for seed in (5, 6, 7):
        nx, ny, _, _ = _inputs(T, 2560, torch.float32, torch.float16, seed=seed)
        x.copy_(nx), y.copy_(ny)
        graph.replay()
        s1, h1 = n(x, y)
        _, r1 = n(x, y, f8=True)
        assert torch.equal(s, s1) and torch.equal(h, h1) and torch.equal(rows.codes.view(torch.uint8), r1.codes.view(torch.uint8))


def test_refusals(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    x, y, w, _ = _inputs(8, 64, torch.float32, torch.float16)
    for code, a, kw in ((-5, (x.cpu(), y), {}), (-5, (x, y.cpu()), {}), (-2, (x, y[:4]), {}), (-2, (x[0], y), {}), (-2, (x.double(), y), {}),
                        (-4, (x.bfloat16(), y), {}), (-4, (x, None), {}), (-4, (x, y), dict(norm="batch")), (-2, (x, y), dict(eps=-1.0)),
                        (-2, (x, y), dict(eps=float("nan"))), (-2, (x, y), dict(alpha=float("inf"))), (-2, (x, y, w[:60]), {}),
                        (-2, (x, y, w.half()), {}), (-3, (x.t().contiguous().t(), y), {}), (-2, (x[:, :60], y[:, :60]), {}),
                        (-3, (x, y), dict(out=y)), (-3, (x.half(), y), dict(sum_out=y)), (-2, (x, y), dict(out=x)),
                        (-2, (x, y), dict(sum_out=y)), (-2, (x.half(), None), dict(alpha=2.0)), (-2, (x.half(), None), dict(sum_out=x.half())),
                        (-3, (x.half(), y), dict(sum_out=x.half()[:1].expand(8, 64)))):
        with pytest.raises(E) as e:
            K.add_norm(*a, **kw)
        assert e.value.code == code, (a, kw, e.value)
    with pytest.raises(E):
        K.add_norm_f8(x[:, :24].contiguous(), y[:, :24].contiguous())  # 16 values at a time
    for bad in (lambda: pkg.norm.AddNorm(w, norm="none"), lambda: pkg.norm.AddNorm(w, w[:3]), lambda: pkg.norm.AddNorm(w)(x[:, :32]),
                lambda: pkg.norm.AddNorm(w)(x, y, f8=True, out=y)):
        with pytest.raises(ValueError):
            bad()
