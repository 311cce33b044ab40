"""The e4m3 linear with block scales against its definition (codes by the same fp32 steps, sums in 64 bits)."""

import math

import pytest
import torch

from oracle import f8 as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _inputs(M, K, N, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * (1 + 20 * (torch.rand(K, generator=g, device=DEV) < 0.02))
    w = torch.randn(N, K, generator=g, device=DEV) / math.sqrt(K)
    return x.to(dtype), w


def _check(y, x, codes, scales):
    ref, bound = O.linear(x, codes, scales)
    worst = float(((y.double() - ref).abs() / bound).max())
    assert worst <= 1.0, f"error {worst:.2f} of its bound"
    # the whole: roundings (half a step u at most each) and cuts, of either sign, add in squares; a cut is at most
    # 2^-13 of the largest of 8 products, 3 to 4 times their spread, so 2^-11 of y's, and both are less on average
    rel = float((y.double() - ref).norm() / ref.norm().clamp_min(1e-30))
    assert rel <= {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[x.dtype] + 2.0 ** -11, rel


@pytest.mark.parametrize("K,N", [(16, 8), (128, 64), (144, 72), (1104, 1608), (2560, 640), (272, 1000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_against_the_definition(gpu_lib, pkg, K, N, dtype):
    for M in (1, 2, 15, 16, 17, 33, 64, 65, 238, 300):
        x, w = _inputs(M, K, N, dtype, seed=M + K)
        lin = pkg.f8.F8Linear.from_float(w)
        buf = torch.full((M * N + 128,), 9.0, dtype=dtype, device=DEV)
        y = pkg.kernels.f8_linear(x, lin.codes_packed, lin.scales, N, out=buf[64:64 + M * N].view(M, N))
        _check(y, x, lin.codes, lin.scales)
        assert bool((buf[:64] == 9.0).all() and (buf[64 + M * N:] == 9.0).all())


@pytest.mark.parametrize("M,K,N", [(1, 272, 8200), (5, 144, 9240), (16, 400, 10240), (16, 2576, 9720), (9, 1040, 4616)])
def test_few_rows_of_wide_outputs(gpu_lib, pkg, M, K, N):
    # (16, 32 and 64 weight rows a workgroup; test_against_the_definition has the narrow ones)
    x, w = _inputs(M, K, N, torch.bfloat16, seed=3)
    lin = pkg.f8.F8Linear.from_float(w)
    _check(lin(x), x, lin.codes, lin.scales)


@pytest.mark.parametrize("M,K,N", [(238, 2560, 7680), (140, 400, 7800), (197, 144, 8000), (100, 1296, 10248), (500, 640, 2560),
                                   (96, 2560, 10240), (90, 272, 9000)])
def test_some_rows_in_tiles_of_128_and_two_rounds(gpu_lib, pkg, M, K, N):
    x, w = _inputs(M, K, N, torch.float16, seed=5)
    lin = pkg.f8.F8Linear.from_float(w)
    buf = torch.full((M * N + 128,), 9.0, dtype=x.dtype, device=DEV)
    y = pkg.kernels.f8_linear(x, lin.codes_packed, lin.scales, N, out=buf[64:64 + M * N].view(M, N))
    _check(y, x, lin.codes, lin.scales)
    assert bool((buf[:64] == 9.0).all() and (buf[64 + M * N:] == 9.0).all())


@pytest.mark.parametrize("M,K,N", [(2049, 272, 8000), (4100, 640, 3584), (1000, 5120, 2560), (3481, 2560, 7680),
                                   (1000, 10240, 2560), (600, 8192, 1024), (530, 2576, 7688), (1010, 2560, 7680)])
def test_many_rows(gpu_lib, pkg, M, K, N):
    x, w = _inputs(M, K, N, torch.bfloat16, seed=1)
    lin = pkg.f8.F8Linear.from_float(w)
    _check(lin(x), x, lin.codes, lin.scales)


@pytest.mark.parametrize("M", [17, 40, 96, 97, 130, 238, 250, 330])
@pytest.mark.parametrize("N", [2560, 7688])
def test_every_tile_height_of_some_rows(gpu_lib, pkg, M, N):
    x, w = _inputs(M, 1168, N, torch.bfloat16, seed=7)
    lin = pkg.f8.F8Linear.from_float(w)
    buf = torch.full((M * N + 128,), 9.0, dtype=x.dtype, device=DEV)
    y = pkg.kernels.f8_linear(x, lin.codes_packed, lin.scales, N, out=buf[64:64 + M * N].view(M, N))
    _check(y, x, lin.codes, lin.scales)
    assert bool((buf[:64] == 9.0).all() and (buf[64 + M * N:] == 9.0).all())


def test_weights_from_float_and_codes(gpu_lib, pkg):
    for N, K in ((8, 16), (200, 400), (640, 256)):
        w = torch.randn(N, K, generator=torch.Generator().manual_seed(N)) * torch.logspace(-3, 3, K)
        w[0, :] = 0
        if N > 128:
            w[128:, :128] = 0  # whole blocks of zeros
        w = w.to(DEV)
        q, s = pkg.kernels.f8_quantize_weight(w)
        qr, sr = O.quantize_weight(w.cpu())  # (IEEE division on both sides)
        assert torch.equal(q.cpu(), qr.view(torch.uint8)) and torch.equal(s.cpu(), sr)
        lin = pkg.f8.F8Linear(qr, sr)
        assert torch.equal(lin.codes.cpu().view(torch.uint8), qr.view(torch.uint8))
        W = lin.dequantized().cpu()
        # a code is half a step (2^-4 of the value) off, or below e4m3's normal range half of 2^-9 scales
        step = sr.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K] * 2.0 ** -10
        assert bool(((W - w.cpu()).abs() <= torch.maximum(w.cpu().abs() * 2.0 ** -4, step) * (1 + 2.0 ** -20)).all())


@pytest.mark.parametrize("M", [3, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_zeros_infinities_and_small_values(gpu_lib, pkg, M, dtype):
    x, w = _inputs(M, 400, 128, dtype)
    x[0] = 0
    x[1, 130] = math.inf
    x[2, 399] = math.nan
    if M > 3:
        x[3] = x[3] * 1e-4
        x[4, :128] = 0
        x[5] = torch.finfo(dtype).max
        x[6] = torch.finfo(dtype).smallest_normal / 4
    lin = pkg.f8.F8Linear.from_float(w)
    y = lin(x)
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    if M > 3:
        for rows in ([3, 4], list(range(7, M))):
            _check(y[rows], x[rows], lin.codes, lin.scales)
        ref, bound = O.linear(x[5:7], lin.codes, lin.scales)
        # near the type's largest value a result may round to it or to infinity; sums whose terms pass fp32's range
        # may end anywhere beyond
        q, s = O.quantize_rows(x[5:7].cpu())
        S = (q * s.double().repeat_interleave(128, 1)[:, :400]).abs() @ lin.dequantized().cpu().double().abs().t()
        fits = (ref.abs() + bound < torch.finfo(dtype).max) & (S.to(DEV) < torch.finfo(torch.float32).max)
        assert bool((((y[5:7].double() - ref).abs() <= bound) | ~fits).all())
        past = ref.abs() - bound > torch.finfo(dtype).max * (1 + 2.0 ** -7)
        assert not bool(torch.isfinite(y[5:7][past]).any())


@pytest.mark.parametrize("M", [1, 16, 238])
def test_views_types_and_shapes(gpu_lib, pkg, M):
    x, w = _inputs(M, 256, 192, torch.float16, seed=4)
    lin = pkg.f8.F8Linear.from_float(w)
    ref = lin(x)
    wide = torch.zeros(M, 640, dtype=torch.float16, device=DEV)
    wide[:, 128:384] = x
    assert torch.equal(lin(wide[:, 128:384]), ref)                      # rows apart, read in place
    assert torch.equal(lin(wide[:, 127:383].clone()[:, 1:][:, :255].new_zeros(M, 256).copy_(x)), ref)
    odd = torch.zeros(M, 257, dtype=torch.float16, device=DEV)
    odd[:, 1:] = x
    assert torch.equal(lin(odd[:, 1:]), ref)                            # misaligned rows: copied first
    assert torch.equal(lin(x.view(1, M, 256)), ref.view(1, M, 192))
    assert torch.equal(lin(x.float()), ref.float())
    assert lin(x[:0]).shape == (0, 192) and lin(x.new_zeros(2, 0, 256)).shape == (2, 0, 192)


@pytest.mark.parametrize("M,K,N", [(1, 2560, 640), (238, 5120, 2560), (2049, 272, 8000), (1000, 10240, 2560)])
def test_partials_sum_to_the_result(gpu_lib, pkg, M, K, N):
    # (one form of each kind; 1000 rows of a long K are split between workgroups)
    x, w = _inputs(M, K, N, torch.float16, seed=2)
    lin = pkg.f8.F8Linear.from_float(w)
    y = lin(x)
    parts, splits = lin.partials(x)
    acc = parts[0].clone()
    for s in range(1, splits):
        acc += parts[s]
    assert torch.equal(acc.half(), y)
    none, one = lin.partials(x[:0])
    assert none.shape == (1, 0, N) and one == 1


@pytest.mark.parametrize("M", [5, 238])
def test_graph_and_repeats(gpu_lib, pkg, M):
    x, w = _inputs(M, 2560, 2560, torch.bfloat16, seed=6)
    lin = pkg.f8.F8Linear.from_float(w)
    ref = lin(x)
    out = torch.empty_like(ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.kernels.f8_linear(x, lin.codes_packed, lin.scales, 2560, out=out)
    keep = pkg.scratch.current(DEV)
    for _ in range(3):
        out.zero_()
        graph.replay()
        again = lin(x)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(again, ref)
    del keep


@pytest.mark.parametrize("M,K,N", [(100, 640, 2560), (1000, 10240, 2560)])
def test_graphs_have_workspaces_of_their_own(gpu_lib, pkg, M, K, N):
    # (the second with partials of a divided K beside x in e4m3)
    lins, xs, graphs, outs, refs = [], [], [], [], []
    for seed in (1, 2):
        x, w = _inputs(M, K, N, torch.bfloat16, seed=seed)
        lin = pkg.f8.F8Linear.from_float(w)
        lins.append(lin), xs.append(x), refs.append(lin(x))
    before = pkg.scratch.generation(DEV)
    for lin, x in zip(lins, xs):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(lin(x))
        graphs.append(graph)
    assert pkg.scratch.generation(DEV) == before
    with pkg.scratch.guard(DEV):
        pkg.scratch.get(pkg.scratch.current(DEV).numel() + 1, DEV).fill_(255)
    side = torch.cuda.Stream()
    for _ in range(5):
        for o in outs:
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(10):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, refs))


def test_codes_that_are_not_numbers(gpu_lib, pkg):
    # a NaN code makes its own output column NaN, nothing else
    x, w = _inputs(40, 256, 192, torch.float16)
    lin = pkg.f8.F8Linear.from_float(w)
    codes = lin.codes.view(torch.uint8).clone()
    codes[70, 33] = 0x7f
    bad = pkg.f8.F8Linear(codes, lin.scales)
    for rows in (x[:3], x):
        y, z = lin(rows), bad(rows)
        cols = [i for i in range(192) if i != 70]
        assert bool(z[:, 70].isnan().all()) and torch.equal(y[:, cols], z[:, cols])


def test_refusals(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    x, w = _inputs(4, 256, 128, torch.float16)
    lin = pkg.f8.F8Linear.from_float(w)

    def refused(code, *a, **kw):
        with pytest.raises(E) as e:
            K.f8_linear(*a, **kw)
        assert e.value.code == code, str(e.value)

    c, s = lin.codes_packed, lin.scales
    refused(-2, x.float(), c, s, 128)
    refused(-5, x.cpu(), c, s, 128)
    refused(-2, x[:, :128], c, s, 128)
    refused(-2, x, c, s, 64)
    refused(-5, x, c.cpu(), s, 128)
    refused(-2, x, c, s.half(), 128)
    refused(-3, x.t()[:, :4].t()[:, ::2], c, s, 128)
    refused(-2, x, c, s, 128, out=torch.empty(4, 64, dtype=torch.float16, device=DEV))
    refused(-2, x, c, s, 128, out=torch.empty(4, 128, dtype=torch.bfloat16, device=DEV))
    square = pkg.f8.F8Linear.from_float(torch.zeros(256, 256, device=DEV))
    refused(-3, x, square.codes_packed, square.scales, 256, out=x)
    refused(-2, x[:, :250].contiguous(), c, s, 128)       # K = 250 rounds to the same pieces: no multiple of 16
    for bad in ((lin.codes[:, :250], s), (lin.codes, s[:, :1]), (lin.codes.float(), s), (lin.codes[:100], s)):
        with pytest.raises(ValueError):
            pkg.f8.F8Linear(*bad)
    with pytest.raises(ValueError):
        lin(x[:, :128])
