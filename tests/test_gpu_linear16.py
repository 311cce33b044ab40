"""The 16-bit linear, and the end that it and the e4m3 linear share, against 64 bits."""

import math
import threading

import pytest
import torch

from oracle import around as O, f8 as O8

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def _inputs(M, K, N, dtype, gated=False, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x = r(M, K) * (1 + 9 * (torch.rand(K, generator=g, device=DEV) < 0.02))
    return x.to(dtype), r(N, K) / math.sqrt(K), r(N), r(M, N // 2 if gated else N).to(dtype)


def _within(y, ref, bound, dtype):
    worst = float(((y.double() - ref).abs() / bound).max())
    assert worst <= 1.0, f"error {worst:.2f} of its bound"


def _check(y, x, w, bias, act, gated, res, alpha):
    z, dz = O.product16(x, w)
    ref, bound = O.end(z, dz, bias, act, gated, res, alpha, x.dtype)
    _within(y, ref, bound, x.dtype)
    # as a whole: roundings of half a step at most add in squares; fp32's sums are far below them
    rel = float((y.double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert rel <= O.HALF_STEP[x.dtype], rel


@pytest.mark.parametrize("K,N", [(8, 8), (64, 64), (72, 72), (136, 1608), (1104, 200), (2560, 640), (640, 2560)])
@pytest.mark.parametrize("dtype", TYPES)
def test_against_the_definition(gpu_lib, pkg, K, N, dtype):
    for i, M in enumerate((1, 2, 15, 16, 17, 33, 64, 65, 150, 238, 300, 700)):
        x, w, b, r = _inputs(M, K, N, dtype, seed=M + K)
        lin = pkg.linear.Linear16.from_float(w, b if i % 2 else None, dtype=dtype)
        res, alpha, act = (r, 0.5, ACTS[i % 5]) if i % 3 == 0 else (None, 1.0, ACTS[i % 5])
        buf = torch.full((M * N + 128,), 9.0, dtype=dtype, device=DEV)
        y = lin(x, act, res, alpha, out=buf[64:64 + M * N].view(M, N))
        _check(y, x, lin.weight, lin.bias, act, False, res, alpha)
        assert bool((buf[:64] == 9.0).all() and (buf[64 + M * N:] == 9.0).all())


@pytest.mark.parametrize("K,N", [(8, 16), (136, 48), (640, 1296), (2560, 10240)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated(gpu_lib, pkg, K, N, dtype):
    for i, M in enumerate((1, 5, 16, 31, 100, 238, 600, 1100)):
        if M * K * N > 1e10 and M > 300:
            continue
        x, w, b, r = _inputs(M, K, N, dtype, gated=True, seed=M)
        lin = pkg.linear.Linear16.from_float(w, b if i % 2 else None, gated=True, dtype=dtype)
        res, act = (r if i % 3 == 0 else None), ACTS[i % 5]
        y = lin(x, act, res, 2.0 if res is not None else 1.0)
        assert y.shape == (M, N // 2) and torch.equal(lin.weight, w.to(dtype))
        _check(y, x, lin.weight, lin.bias, act, True, res, 2.0 if res is not None else 1.0)


@pytest.mark.parametrize("M,K,N", [(1, 2560, 10240), (16, 8192, 4096), (7, 5120, 2560), (4, 100 * 8, 8200), (238, 5120, 2560),
                                   (238, 2560, 7680), (512, 5120, 2560), (1000, 2560, 2560), (1000, 10240, 2560), (2049, 1104, 1608),
                                   (3481, 640, 2560), (4100, 640, 3584), (600, 8192, 1024), (90, 272, 9000), (1500, 2576, 7688)])
def test_every_form(gpu_lib, pkg, M, K, N):
    x, w, b, _ = _inputs(M, K, N, torch.bfloat16, seed=1)
    lin = pkg.linear.Linear16.from_float(w, b, dtype=torch.bfloat16)
    _check(lin(x, "silu"), x, lin.weight, lin.bias, "silu", False, None, 1.0)


@pytest.mark.parametrize("M", [3, 40, 700])
def test_rows_apart_and_the_residual_in_place(gpu_lib, pkg, M):
    x, w, _, r = _inputs(M, 640, 320, torch.float16)
    lin = pkg.linear.Linear16.from_float(w)
    want = lin(x, residual=r)
    wide = torch.full((M, 1928), float("nan"), dtype=torch.float16, device=DEV)  # what lies beside rows is not read
    wide[:, 640:1280] = x
    assert torch.equal(lin(wide[:, 640:1280], residual=r), want)
    apart = torch.full((M, 648), float("nan"), dtype=torch.float16, device=DEV)
    apart[:, 8:328] = r
    assert torch.equal(lin(x, residual=apart[:, 8:328]), want)
    one = x[:1].expand(M, 640)
    assert torch.equal(lin(one), lin(one.contiguous()))
    odd = torch.empty(M * 640 + 1, dtype=torch.float16, device=DEV)[1:].view(M, 640)
    odd.copy_(x)
    assert torch.equal(lin(odd, residual=r), want) and torch.equal(lin(x.t().contiguous().t(), residual=r), want)
    assert torch.equal(lin(x.view(1, M, 640), residual=r.view(1, M, 320)), want.view(1, M, 320))
    kept = r.clone()
    assert lin(x, residual=kept, out=kept).data_ptr() == kept.data_ptr() and torch.equal(kept, want)


@pytest.mark.parametrize("M", [9, 100, 700])
def test_a_rows_nan_stays_in_its_row(gpu_lib, pkg, M):
    x, w, b, _ = _inputs(M, 200, 320, torch.bfloat16)
    lin = pkg.linear.Linear16.from_float(w, b, dtype=torch.bfloat16)
    want = lin(x, "gelu")
    bad = x.clone()
    bad[M // 2, 3], bad[0, 199] = float("nan"), float("inf")
    y = lin(bad, "gelu")
    same = [i for i in range(M) if i not in (0, M // 2)]
    assert torch.equal(y[same], want[same]) and bool(y[M // 2].isnan().all()) and not bool(torch.isfinite(y[0]).any())


def test_activations_far_out(gpu_lib, pkg):
    z = torch.tensor([0.0, -0.0, 1e-6, -1e-6, 0.5, -0.5, 3, -3, 6, -6, 12, -12, 40, -40, 90, -90, 1000, -1000, 30000, -30000, 60000, -60000,
                      float("inf"), float("nan")], device=DEV)
    x = torch.zeros(1, 8, dtype=torch.float16, device=DEV)
    w = torch.zeros(24, 8, device=DEV)
    for act in ACTS:
        lin = pkg.linear.Linear16.from_float(w, z)
        y = lin(x, act)[0]
        ref, bound = O.end(torch.zeros(1, 24, device=DEV).double(), torch.zeros(1, 24, device=DEV).double(), z, act, False, None, 1.0, torch.float16)
        ref, bound = ref[0], bound[0]
        assert bool(((y[:22].double() - ref[:22]).abs() <= bound[:22]).all()), act
        assert float(y[22]) == math.inf and bool(y[23].isnan())


@pytest.mark.parametrize("M,K,N", [(5, 2560, 2560), (238, 5120, 2560), (1000, 10240, 2560)])
def test_captured_and_replayed(gpu_lib, pkg, M, K, N):
    x, w, b, r = _inputs(M, K, N, torch.bfloat16)
    lin = pkg.linear.Linear16.from_float(w, b, dtype=torch.bfloat16)
    lin(x, "gelu", r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x, "gelu", r)
    pkg.scratch.release()  # (the graph's workspace is its own)
    for seed in (4, 5, 6):
        x.copy_(_inputs(M, K, N, torch.bfloat16, seed=seed)[0])
        graph.replay()
        assert torch.equal(y, lin(x, "gelu", r))


def test_two_threads_on_their_own_streams(gpu_lib, pkg):
    x, w, b, r = _inputs(1000, 10240, 2560, torch.bfloat16)  # K is split: both use the scratch
    lin = pkg.linear.Linear16.from_float(w, b, dtype=torch.bfloat16)
    assert pkg.capi.lib().linear16_workspace_bytes(1000, 10240, 2560, 0) > 0
    want = [lin(x, "silu"), lin(x, residual=r)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                y = lin(x, "silu") if i == 0 else lin(x, residual=r)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    x, w, b, r = _inputs(8, 64, 48, torch.float16)
    lin = pkg.linear.Linear16.from_float(w, b)
    p, n = lin.packed, 48
    call = lambda *a, **kw: K.linear16(*a, **kw)  # noqa: E731
    for code, a, kw in ((-5, (x.cpu(), p, n), {}), (-2, (x.float(), p, n), {}), (-2, (x[0], p, n), {}), (-2, (x[:, :60], p, n), {}),
                        (-2, (x, p, 40 * 8), {}), (-2, (x, p.view(torch.int32), n), {}), (-2, (x, p, n, b[:40]), {}), (-2, (x, p, n, b.half()), {}),
                        (-4, (x, p, n), dict(activation="tanh")), (-2, (x, p, n), dict(residual=r[:4])), (-2, (x, p, n), dict(residual=r.float())),
                        (-2, (x, p, n), dict(alpha=float("nan"))), (-3, (x.t().contiguous().t(), p, n), {}), (-2, (x, p, n), dict(out=r[:4])),
                        (-3, (x, p, n), dict(residual=r[:1].expand(8, 48))), (-3, (x[:, 4:60], K.linear16_pack(w[:, 4:60].half().contiguous()), n), {}),
                        (-5, (x, p, n), dict(out=r.cpu())), (-3, (x[:, :48].contiguous(),) * 2, {})):
        if len(a) == 2:  # out over x
            y = a[0]
            a, kw = (y, K.linear16_pack(w[:, :48].half().contiguous()), n), dict(out=y)
        with pytest.raises(E) as e:
            call(*a, **kw)
        assert e.value.code == code, (code, kw, e.value)
    for bad in (lambda: pkg.linear.Linear16(w), lambda: pkg.linear.Linear16(w[:, :60].half()), lambda: pkg.linear.Linear16(w[:44].half()),
                lambda: pkg.linear.Linear16(w[:40].half(), gated=True), lambda: pkg.linear.Linear16(w.half(), b[:3]), lambda: lin(x[:, :32]),
                lambda: lin(x.bfloat16()), lambda: lin(x, residual=r[:4])):
        with pytest.raises(ValueError):
            bad()
    assert lin(x[:0]).shape == (0, 48) and lin(x[:0], "gelu", r[:0]).shape == (0, 48)


# ---- the same end on e4m3 weights ------------------------------------------------------------------
def _check8(y, xd, lin, bias, act, res, alpha, dtype):
    z, dz = O.product8(xd, lin.codes, lin.scales)
    ref, bound = O.end(z, dz, bias, act, lin.gated, res, alpha, dtype)
    _within(y, ref, bound, dtype)


def _quantized(x):
    q, s = O8.quantize_rows(x.cpu())
    return (q * s.double().repeat_interleave(128, 1)[:, :x.shape[1]]).to(x.device)


@pytest.mark.parametrize("K,N,gated", [(16, 8, False), (144, 64, True), (1104, 1608, False), (2560, 640, False), (272, 1280, True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_e4m3_with_an_end(gpu_lib, pkg, K, N, gated, dtype):
    for i, M in enumerate((1, 9, 16, 17, 40, 100, 238, 700)):
        x, w, b, r = _inputs(M, K, N, dtype, gated, seed=M + K)
        lin = pkg.f8.F8Linear.from_float(w, bias=b if i % 2 else None, gated=gated)
        res, act, alpha = (r if i % 3 == 0 else None), ACTS[i % 5], 1.5
        _check8(lin(x, act, res, alpha), _quantized(x), lin, b if i % 2 else None, act, res, alpha, dtype)
        # and from rows that the norm left in e4m3
        n = pkg.norm.AddNorm(torch.ones(K))
        _, rows = n(x, f8=True)
        y = lin(rows, act, res, alpha)
        assert y.dtype is dtype
        _check8(y, rows.dequantized().double(), lin, b if i % 2 else None, act, res, alpha, dtype)


@pytest.mark.parametrize("M,K,N,gated", [(1, 2560, 10240, True), (16, 5120, 2560, False), (238, 5120, 2560, False), (238, 2560, 7680, True),
                                         (1000, 10240, 2560, False), (3481, 2560, 2560, True), (2049, 272, 8000, False), (500, 640, 2560, True)])
def test_e4m3_every_form(gpu_lib, pkg, M, K, N, gated):
    x, w, b, _ = _inputs(M, K, N, torch.bfloat16, gated, seed=2)
    lin = pkg.f8.F8Linear.from_float(w, bias=b, gated=gated)
    _check8(lin(x, "silu"), _quantized(x), lin, b, "silu", None, 1.0, torch.bfloat16)
    _, rows = pkg.norm.AddNorm(torch.ones(K))(x, f8=True)
    _check8(lin(rows, "silu"), rows.dequantized().double(), lin, b, "silu", None, 1.0, torch.bfloat16)


@pytest.mark.parametrize("M", [4, 100, 1000])
def test_e4m3_gives_back_its_weights_and_the_bits_without_an_end(gpu_lib, pkg, M):
    x, w, _, _ = _inputs(M, 640, 384, torch.float16)
    plain, gated = pkg.f8.F8Linear.from_float(w), pkg.f8.F8Linear.from_float(w, gated=True)
    assert torch.equal(plain.codes.view(torch.uint8), gated.codes.view(torch.uint8)) and torch.equal(plain.dequantized(), gated.dequantized())
    y = pkg.kernels.f8_linear_end(x, plain.codes_packed, plain.scales, 384)
    assert torch.equal(y, plain(x))
    z = gated(x)  # no activation: g u, of the products before their rounding
    ref, bound = (plain(x).double()[:, :192] * plain(x).double()[:, 192:]), None
    assert float((z.double() - ref).norm() / ref.norm()) <= 3 * 2.0 ** -11
    with pytest.raises(ValueError):
        gated.partials(x)
    with pytest.raises(ValueError):
        pkg.f8.F8Linear.from_float(w[:360], gated=True)
    with pytest.raises(ValueError):
        plain(pkg.norm.AddNorm(torch.ones(320))(x[:, :320].contiguous(), f8=True)[1])


def test_e4m3_rows_captured(gpu_lib, pkg):
    x, w, b, r = _inputs(1000, 5120, 2560, torch.bfloat16)
    lin, n = pkg.f8.F8Linear.from_float(w, bias=b), pkg.norm.AddNorm(torch.ones(5120))
    run = lambda: lin(n(x, f8=True)[1], "gelu_tanh", r)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for seed in (4, 5, 6):
        x.copy_(_inputs(1000, 5120, 2560, torch.bfloat16, seed=seed)[0])
        graph.replay()
        assert torch.equal(y, run())
