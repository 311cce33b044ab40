"""Edges of the residual's norm, the linears with an end and the cache in 4 bits that their first tests do not reach."""

import pytest
import torch

from oracle import around as A, cache4 as C4
from test_gpu_cache4 import Case
from test_gpu_esmc_packed import _gen
from test_gpu_linear16 import _inputs
from test_gpu_norm import _check as check_norm, _check8 as check_norm8, _inputs as norm_inputs
from test_gpu_together import _hf

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


@pytest.mark.parametrize("nq,nk,H,Hk,d", [([1], [9000], 32, 8, 128), ([1] * 8, [16385, 9002, 4097, 2501, 1025, 334, 77, 1], 32, 8, 128),
                                          ([5, 40], [3000, 700], 16, 2, 64), ([200], [900], 10, 10, 80)])
@pytest.mark.parametrize("dtype", TYPES)
def test_probabilities_keep_16_bits(gpu_lib, pkg, nq, nk, H, Hk, d, dtype):
    """The output's rounding is what there is to see. A kernel that holds o + e, |e| <= E, and rounds once is off by at most
    the distance of o + e from the nearest value of the type, so by |round(o) - o| + 2 E at most; E is the oracle's bound
    with probability times step kept to 2^-16, whatever the type, and without the rounding of o."""
    c = Case(pkg, nq, nk, H, Hk, d, dtype, seed=3).fill()
    o = c.attend().double()
    held = [C4.hold(t) for t in (c.k, c.v)]
    off = least = size = 0.0
    for i in range(len(nq)):
        rows, keys = slice(c.cq[i], c.cq[i + 1]), slice(c.ck[i], c.ck[i + 1])
        ref, bound = C4.attention(c.q[rows], *([t[keys] for t in h] for h in held), True, d ** -0.5, u_p=2.0 ** -16)
        E = bound - A.HALF_STEP[dtype] * ref.abs() - A.SMALLEST[dtype]
        once = (ref.to(dtype).double() - ref).abs()
        worst = float(((o[rows] - ref).abs() / (once + 2 * E + A.SMALLEST[dtype])).max())
        assert worst <= 1.0, f"sequence {i}: {worst:.2f} of one rounding and 16 bits of the probabilities"
        off, least, size = off + (o[rows] - ref).pow(2).sum(), least + once.pow(2).sum(), size + ref.pow(2).sum()
    # As a whole: the scores' roundings, of magnitudes some 1,000 times a value of q, make p off by 2^-16 or so, P's own are
    # 2^-17, independent from key to key; fp16's rounding of o is 2^-12.2, eleven times their sum, and 1.05 leaves room for
    # 0.32 of it beside it in squares.
    assert float(off) <= 1.05 ** 2 * float(least), f"{float((off / size) ** 0.5):.2e} off, one rounding {float((least / size) ** 0.5):.2e}"


def test_outputs_that_lie_on_an_operand_elsewhere_than_at_its_start(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    for T in (5, 1100):
        buf = torch.randn(T + 9, 192, device=DEV).half()
        x, y, w = buf[:T, :64], torch.randn(T, 64, device=DEV).half(), torch.ones(64, device=DEV)
        ybuf = torch.zeros(T + 1, 64, dtype=torch.float16, device=DEV)
        wide = torch.zeros(T + 1, 64, dtype=torch.float32, device=DEV)
        for kw in (dict(sum_out=buf[1:T + 1, :64]), dict(sum_out=buf[:T, 8:72]), dict(out=buf[1:T + 1, :64]), dict(out=buf[:T, 56:120]),
                   dict(sum_out=buf[:T, 64:128], out=buf[2:T + 2, 64:128])):
            with pytest.raises(E) as e:
                K.add_norm(x, y, w, **kw)
            assert e.value.code == -3, kw
        with pytest.raises(E):
            K.add_norm(x, ybuf[:T], w, out=ybuf[1:])
        with pytest.raises(E):
            K.add_norm(wide[:T], y, wide[T], sum_out=wide[1:])  # over the weight
        s, h = K.add_norm(x.clone(), y, w)
        s1, h1 = K.add_norm(x, y, w, sum_out=buf[:T, 64:128], out=buf[:T, 128:])  # beside x in its rows
        assert torch.equal(s, s1) and torch.equal(h, h1)
        s1, h1 = K.add_norm(x, y, w, sum_out=x, out=buf[:T, 128:])
        assert torch.equal(s, s1) and torch.equal(h, h1)
    x = torch.randn(40, 64, device=DEV).half()
    lin = pkg.linear.Linear16.from_float(torch.randn(64, 64, device=DEV), torch.randn(64, device=DEV))
    r = torch.randn(41, 64, device=DEV).half()
    e8 = pkg.f8.F8Linear.from_float(torch.randn(64, 64, device=DEV))
    for call in (lambda: lin(x[:32], out=x[8:]), lambda: lin(x[:39], residual=r[:39], out=r[1:40]), lambda: lin(x[8:], out=x.view(-1)[504:504 + 2048]),
                 lambda: K.f8_linear_end(x[:32], e8.codes_packed, e8.scales, 64, out=x[8:]), lambda: K.f8_linear(x[:32], e8.codes_packed, e8.scales, 64, out=x[8:])):
        with pytest.raises(E) as e:
            call()
        assert e.value.code == -3
    want = lin(x[:39], residual=r[:39])
    assert torch.equal(lin(x[:39], residual=r[:39], out=r[:39]), want)
    both = torch.randn(80, 64, device=DEV).half()
    assert torch.equal(lin(both[:40], out=both[40:]), lin(both[:40].clone()))
    c = Case(pkg, [5, 60], [200, 100], 8, 2, 64, torch.bfloat16).fill()
    want, wide = c.attend(), torch.zeros(66, 24, 64, dtype=torch.bfloat16, device=DEV)
    wide[:65, :8] = c.q
    q = wide[:65, :8]
    for out in (wide[1:, :8], wide[:65, 4:12], wide[:65, 7:15]):
        with pytest.raises(E) as e:
            c.cache.attend(q, c.cu, c.lens, c.table, out=out)
        assert e.value.code == -3
    assert torch.equal(c.cache.attend(q, c.cu, c.lens, c.table, out=wide[:65, 8:16]), want)
    cu = torch.tensor([0, 65], dtype=torch.int32, device=DEV)
    q, k, v = wide[:65, :8], wide[:65, 8:16], wide[:65, 16:]
    for out in (wide[1:, :8], wide[1:, 8:16], wide[:65, 12:20], wide[1:, 16:]):
        with pytest.raises(E) as e:
            K.packed_attention(q, k, v, cu, out=out)
        assert e.value.code == -3
    freq = torch.ones(32, dtype=torch.float64, device=DEV)
    for out in ((wide[1:, :8], k), (q, wide[1:, 8:16]), (k, q), (wide[:65, 4:12], wide[:65, 16:])):
        with pytest.raises(E) as e:
            K.qk_norm_rope(q, k, freq, out=out)
        assert e.value.code == -3
    one = wide[:65, 0, :].contiguous().view(-1)  # a head each, the second half a head further
    with pytest.raises(E):
        K.qk_norm_rope(one[:4096].view(64, 1, 64), one[32:4128].view(64, 1, 64), freq, out=(one[:4096].view(64, 1, 64), one[32:4128].view(64, 1, 64)))
    want = K.qk_norm_rope(q, k, freq)
    assert all(torch.equal(a, b) for a, b in zip(want, K.qk_norm_rope(q, k, freq, out=(q, k))))


def test_leading_dimensions_of_the_norms_operands_agree(gpu_lib, pkg):
    n = pkg.norm.AddNorm(torch.ones(64))
    x, y = torch.randn(2, 3, 64, device=DEV), torch.randn(2, 3, 64, device=DEV).half()
    h = torch.empty_like(y)
    for call in (lambda: n(x, y.view(3, 2, 64)), lambda: n(x, y.view(6, 64)), lambda: n(x, y, out=h.view(3, 2, 64)), lambda: n(x, y, sum_out=torch.empty(6, 64, device=DEV)),
                 lambda: n(x, y.view(3, 2, 64), f8=True)):
        with pytest.raises(ValueError):
            call()
    s, got = n(x, y, sum_out=x, out=h)
    assert got.data_ptr() == h.data_ptr() and s.data_ptr() == x.data_ptr() and s.shape == got.shape == (2, 3, 64)


def test_values_up_to_the_limit(gpu_lib, pkg):
    c = Case(pkg, [2, 30], [900, 200], 8, 2, 128, torch.bfloat16)
    c.v = (c.v.float().clamp(-4, 4) * 2.0 ** 93.9).to(torch.bfloat16)  # below 2^96
    # a row whose first key is the least, so that what it is made relative to lags behind: p up to 2^8
    c.q[0], c.k[:, :] = 1.0, c.k * 0.01
    c.k[1:900] += 0.04
    c.fill()
    o = c.attend()
    assert bool(torch.isfinite(o).all())
    c.check(o)
    rk, rv = c.cache.read(c.whole, c.lens, c.table)
    assert bool(torch.isfinite(rv).all())
    c.v *= 2.0 ** 30  # held and read as any other
    c.fill()
    for got, x in zip(c.cache.read(c.whole, c.lens, c.table), (c.k, c.v)):
        code, s, z = C4.hold(x)
        assert torch.equal(got, (s * (code - z)).to(torch.bfloat16))


@pytest.mark.parametrize("T", [1, 5, 17, 1023, 1030])  # a row a workgroup, and several
@pytest.mark.parametrize("D", [144, 2560])
def test_what_lies_behind_the_norms_last_row_stays(gpu_lib, pkg, T, D):
    x, y, w, _ = norm_inputs(T, D, torch.float32, torch.bfloat16, seed=T)
    s, h = torch.full((T + 40, D), 7.0, device=DEV), torch.full((T + 40, D), 7.0, dtype=torch.bfloat16, device=DEV)
    pkg.kernels.add_norm(x, y, w, sum_out=s[20:T + 20], out=h[20:T + 20])
    for t in (s, h):
        assert bool((t[:20] == 7).all() and (t[T + 20:] == 7).all())
    check_norm(s[20:T + 20], h[20:T + 20], x, y, 1.0, w, None, "rms", 1e-6)
    # e4m3: blocks of 16 rows, of which the last is not whole
    mp, kb = -(-T // 16) * 16, -(-D // 128)
    n, m = gpu_lib.f8_rows_bytes(T, D), gpu_lib.f8_rows_scales_bytes(T, D)
    assert n == mp * kb * 128 and m == mp * kb * 4 + 1024
    hq, hs = torch.full((n + 4096,), 165, dtype=torch.uint8, device=DEV), torch.full((m // 4 + 1024,), -3.0, device=DEV)
    assert gpu_lib.add_norm(x.data_ptr(), 1, y.data_ptr(), 1.0, s[20:].data_ptr(), None, hq.data_ptr(), hs.data_ptr(), w.data_ptr(), None, 1e-6, 1, D, D, D,
                            0, T, D, 1, pkg.capi.stream_ptr()) == 0
    assert bool((hq[n:] == 165).all() and (hs[kb * mp:] == -3).all())
    behind = hq[:n].view(mp // 16, kb, 2, 4, 16, 16).permute(0, 4, 1, 3, 2, 5).reshape(mp, -1)[T:]
    assert bool((behind == 165).all() and (hs[:kb * mp].view(kb, mp)[:, T:] == -3).all())
    rows = pkg.f8.F8Rows(hq[:n], hs[:m // 4], (T,), D, torch.bfloat16)
    check_norm8(rows, x, y, 1.0, w, None, "rms", 1e-6)
    assert bool((s[:20] == 7).all() and (s[T + 20:] == 7).all())


@pytest.mark.parametrize("D", [8200, 12800, 16904, 20000, 24576, 32768])  # 3 to 11 waves a row, 3 to 8 pieces a lane
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_many_long_rows(gpu_lib, pkg, D, norm):
    for T, stream, dtype in ((1024, torch.float32, torch.float16), (1500, torch.bfloat16, torch.bfloat16)):
        x, y, w, b = norm_inputs(T, D, stream, dtype, seed=D)
        b = b if norm == "layer" else None
        s, h = pkg.kernels.add_norm(x, y, w, b, norm=norm, eps=1e-5)
        check_norm(s, h, x, y, 1.0, w, b, norm, 1e-5)
        if D % 16 == 0:
            _, rows = pkg.norm.AddNorm(w, b, norm=norm, eps=1e-5)(x, y, f8=True)
            check_norm8(rows, x, y, 1.0, w, b, norm, 1e-5)


def test_rows_in_e4m3_of_another_count_are_refused(gpu_lib, pkg, monkeypatch):
    """The scales of a block of columns lie a whole count of 16 rows behind one another: of another, others' would be read."""
    K, lin = pkg.kernels, pkg.f8.F8Linear.from_float(torch.randn(64, 640, device=DEV))
    x = torch.randn(40, 640, device=DEV).half()
    q, s = K.add_norm_f8(x)[1]
    call = lambda M, K_=640: K.f8_linear_end(None, lin.codes_packed, lin.scales, 64, rows=(q, s, M, K_), dtype=torch.float16)  # noqa: E731
    want = call(40)
    for _ in range(2):
        for M, K_ in ((30, 640), (49, 640), (16, 640), (0, 640), (-1, 640), (40, 512)):
            with pytest.raises(pkg.capi.EsmError) as e:
                call(M, K_)
            assert e.value.code == -2, (M, K_)
        assert torch.equal(call(33), want[:33]) and torch.equal(call(40), want)
        monkeypatch.setattr(pkg.capi, "bind", pkg.capi._LongWay)


def test_a_linear_with_another_forward_takes_16_bit_rows(gpu_lib, pkg, monkeypatch):
    """A forward put in the place of a linear's own is written for tensors: the block then runs its separate calls."""
    F8 = pkg.f8.F8Linear
    model = pkg.esmc.HipEsmc.from_hf(_hf(256, 384, 2, 5), n_heads=4, linear=F8, fused=True)
    ids, cu = torch.randint(0, 33, (150,), generator=_gen(3)).to(DEV), torch.tensor([0, 100, 150], dtype=torch.int32, device=DEV)
    want = model.packed_hidden_states(ids, cu)
    blk, seen = model.layers[1], []
    own = blk.wqkv.forward
    blk.wqkv.forward = lambda x: seen.append(x.dtype) or own(x)  # (x.dtype of a tensor)
    assert not blk.takes_rows()
    other = model.packed_hidden_states(ids, cu)
    assert seen == [torch.float16] and float((other[-1] - want[-1]).pow(2).mean().sqrt()) <= 0.15  # (e4m3's error of both)
    del blk.wqkv.forward
    assert blk.takes_rows() and torch.equal(model.packed_hidden_states(ids, cu), want)
    kinds, forward = [], F8.forward
    monkeypatch.setattr(F8, "forward", lambda self, x, *a, **k: kinds.append(type(x)) or forward(self, x, *a, **k))
    assert not blk.takes_rows()
    model.packed_hidden_states(ids, cu)
    assert kinds and all(k is torch.Tensor for k in kinds)


def test_values_next_to_the_types_largest(gpu_lib, pkg):
    c = Case(pkg, [1], [70], 1, 1, 64, torch.float16)
    c.k[5] = torch.linspace(0, 65504, 64, device=DEV).half()  # 15 steps are 65760
    c.v[9] = torch.linspace(-65504, 65504, 64, device=DEV).half()
    c.fill()
    for got, x in zip(c.cache.read(c.whole, c.lens, c.table), (c.k, c.v)):
        code, s, z = C4.hold(x)
        held = s * (code - z)
        assert torch.equal(got, held.half()) and float(((held - x.double()).abs() / s).max()) <= 0.5
    assert bool(c.cache.read(c.whole, c.lens, c.table)[0][5].isinf().any())
