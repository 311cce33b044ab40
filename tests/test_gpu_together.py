"""The residual's norm, the linears with an end and the cache in 4 bits as they are used together: steps of generation, the
packed language model on e4m3 rows; and each call by the native short way as by the longer one."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import around as O, cache4 as C4, esmc as oe, f8 as of8
from test_gpu_cache4 import Case, i32
from test_gpu_esmc_packed import LINEARS, _gen, _weights
from test_gpu_linear16 import _check as check_linear16
from test_gpu_norm import _check8

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Layer:
    """A block that generates: norm -> qkv in e4m3 -> cache and attention on it -> o-projection onto the residual -> norm ->
    gated linear -> down-projection."""

    def __init__(self, pkg, D, Fd, H, Hk, d, dtype, sequences, width):
        g = torch.Generator(device=DEV).manual_seed(D)
        r = lambda n, k: torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)  # noqa: E731
        self.dtype, self.H, self.Hk, self.d = dtype, H, Hk, d
        self.n1, self.n2 = (pkg.norm.AddNorm(1 + 0.1 * torch.randn(D, generator=g, device=DEV)) for _ in range(2))
        self.qkv = pkg.f8.F8Linear.from_float(r((H + 2 * Hk) * d, D), bias=0.1 * torch.randn((H + 2 * Hk) * d, generator=g, device=DEV))
        self.wo = pkg.linear.Linear16.from_float(r(D, H * d), dtype=dtype)
        self.up = pkg.f8.F8Linear.from_float(r(2 * Fd, D), gated=True)
        self.down = pkg.linear.Linear16.from_float(r(D, Fd), dtype=dtype)
        self.cache = pkg.cache4.Cache4(sequences * width, Hk, d, dtype=dtype)
        self.table = torch.randperm(sequences * width, generator=g, device=DEV).int().view(sequences, width)

    def __call__(self, x, y, cu, lens):
        """x the residual (fp32), y what the layer before adds to it. Everything that is made on the way."""
        s1, h1 = self.n1(x, y, f8=True)
        qkv = self.qkv(h1)
        q, k, v = qkv.view(len(x), self.H + 2 * self.Hk, self.d).split([self.H, self.Hk, self.Hk], 1)
        self.cache.append(k, v, cu, lens, self.table)
        o = self.cache.attend(q, cu, lens, self.table)
        a = self.wo(o.view(len(x), -1))
        s2, h2 = self.n2(s1, a, f8=True)
        m = self.up(h2, activation="silu")
        return s1, h1, qkv, o, a, s2, h2, m, self.down(m, residual=a)


def _check_step(layer, got, x, y, cu, lens, keys, values):
    s1, h1, qkv, o, a, s2, h2, m, out = got
    _check8(h1, x, y, 1.0, layer.n1.weight, None, "rms", layer.n1.eps)
    z, dz = O.product8(h1.dequantized().double(), layer.qkv.codes, layer.qkv.scales)
    ref, bound = O.end(z, dz, layer.qkv.bias, None, False, None, 1.0, layer.dtype)
    assert bool(((qkv.double() - ref).abs() <= bound).all())
    H, Hk = layer.H, layer.Hk
    q, k, v = qkv.view(len(x), H + 2 * Hk, layer.d).split([H, Hk, Hk], 1)
    for i, n in enumerate(lens.tolist()):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        keys[i], values[i] = torch.cat([keys[i], k[rows]]), torch.cat([values[i], v[rows]])
        assert len(keys[i]) == n
        ref, bound = C4.attention(q[rows], C4.hold(keys[i]), C4.hold(values[i]), True, layer.d ** -0.5)
        assert bool(((o[rows].double() - ref).abs() <= bound).all()), i
    check_linear16(a, o.view(len(x), -1), layer.wo.weight, None, None, False, None, 1.0)
    _check8(h2, s1, a, 1.0, layer.n2.weight, None, "rms", layer.n2.eps)
    z, dz = O.product8(h2.dequantized().double(), layer.up.codes, layer.up.scales)
    ref, bound = O.end(z, dz, None, "silu", True, None, 1.0, layer.dtype)
    assert bool(((m.double() - ref).abs() <= bound).all())
    check_linear16(out, m, layer.down.weight, None, None, False, a, 1.0)


@pytest.mark.parametrize("D,Fd,H,Hk,d,dtype", [(256, 320, 8, 2, 64, torch.bfloat16), (640, 1280, 10, 10, 64, torch.float16),
                                               (1024, 1024, 8, 1, 128, torch.bfloat16)])
def test_prompts_and_captured_steps(gpu_lib, pkg, D, Fd, H, Hk, d, dtype):
    prompts = [70, 1, 130]
    layer = Layer(pkg, D, Fd, H, Hk, d, dtype, 3, 4)
    g = _gen(7)
    rows = lambda n: (torch.randn(n, D, generator=g).to(DEV), (0.3 * torch.randn(n, D, generator=g)).to(dtype).to(DEV))  # noqa: E731
    keys = [torch.empty(0, Hk, d, dtype=dtype, device=DEV) for _ in prompts]
    values = [t.clone() for t in keys]
    cu = i32(*[sum(prompts[:i]) for i in range(4)])
    lens = i32(*prompts)
    x, y = rows(sum(prompts))
    _check_step(layer, layer(x, y, cu, lens), x, y, cu, lens, keys, values)
    # then a row each, recorded once: lengths and rows change in place
    cu = i32(0, 1, 2, 3)
    x, y = rows(3)
    held = layer.cache.data.clone()
    lens += 1
    layer(x, y, cu, lens)  # (the scratch is there, as in any program)
    layer.cache.data.copy_(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x, y, cu, lens)
    keep = pkg.scratch.current(DEV)
    for step in range(5):
        before = layer.cache.data.clone()
        graph.replay()
        torch.cuda.synchronize()
        _check_step(layer, got, x, y, cu, lens, keys, values)
        after = layer.cache.data.clone()
        layer.cache.data.copy_(before)
        again = layer(x, y, cu, lens)  # the program's own work between the replays, to the bit the same
        assert all(torch.equal(a, b) for a, b in zip(got, again) if isinstance(a, torch.Tensor))
        assert torch.equal(layer.cache.data, after)
        x2, y2 = rows(3)
        x.copy_(x2)
        y.copy_(y2)
        lens += 1
    del keep


def _hf(D, F_, n, seed):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    hf = {"esmc.embed_tokens.weight": r(33, D), "esmc.norm.weight": 1 + 0.1 * r(D)}
    for i in range(n):
        at = f"esmc.layers.{i}."
        for name, shape in {"self_attn.q_proj": (D, D), "self_attn.k_proj": (D, D), "self_attn.v_proj": (D, D), "self_attn.o_proj": (D, D),
                            "mlp.gate_proj": (F_, D), "mlp.up_proj": (F_, D), "mlp.down_proj": (D, F_)}.items():
            hf[f"{at}{name}.weight"] = r(*shape) * shape[1] ** -0.5
        for name in ("input_layernorm", "post_attention_layernorm"):
            hf[f"{at}{name}.weight"], hf[f"{at}{name}.bias"] = 1 + 0.1 * r(D), 0.1 * r(D)
        for name in ("q_norm", "k_norm"):
            hf[f"{at}self_attn.{name}.weight"] = 1 + 0.1 * r(D)
    return hf


@pytest.mark.parametrize("D,F_,H,lengths", [(256, 384, 4, [29, 1, 70, 0, 133]), (640, 640, 10, [200, 65]), (128, 96, 2, [5])])
def test_packed_language_model_on_e4m3_rows(gpu_lib, pkg, D, F_, H, lengths):
    """Part by part, each from what the model gave it: a code that falls to the other side of a border shifts its row by a
    hundredth or so, and then a tenth of the row's next codes, so a bound on a whole block would say little."""
    model = pkg.esmc.HipEsmc.from_hf(_hf(D, F_, 3, 5), n_heads=H, linear=pkg.f8.F8Linear, fused=True)
    assert all(b.takes_rows() for b in model.layers)
    seen = []
    keep = lambda t: t.clone() if isinstance(t, torch.Tensor) else t  # noqa: E731 (the rotation works in place)
    for blk in model.layers:
        for name in LINEARS:
            getattr(blk, name).register_forward_hook(lambda m, args, y: seen.append((m, args[0], keep(y))))
    seqs = [torch.randint(0, 33, (L,), generator=_gen(2)) for L in lengths]
    ids = torch.cat(seqs).to(DEV)
    hs = model.packed([t.to(DEV) for t in seqs]).hidden_states
    assert torch.equal(hs[0], model.embed[ids]) and len(seen) == 12
    alpha = 1.0 / model.res_scale

    def product(at, name, activation=None):
        m, x, y = seen[at]
        assert m is getattr(model.layers[at // 4], name)
        if isinstance(x, torch.Tensor):
            q, scales = of8.quantize_rows(x.cpu())
            x = (q * scales.double().repeat_interleave(128, 1)[:, :x.shape[1]]).to(DEV)
        else:
            x = x.dequantized().double()
        ref, bound = O.end(*O.product8(x, m.codes, m.scales), None, activation, m.gated, None, 1.0, torch.float16)
        assert bool(((y.double() - ref).abs() <= bound).all()), (at, name)
        return y

    for i, blk in enumerate(model.layers):
        at = 4 * i
        _check8(seen[at][1], hs[i], None, 0.0, blk.ln1_w, blk.ln1_b, "layer", 1e-5) if i == 0 else None
        qkv, o = product(at, "wqkv").double().cpu(), seen[at + 1][1].double().cpu()
        q, k, v = qkv.split(D, 1)
        q, k = (F.layer_norm(t, (D,), w.double().cpu(), None, 1e-5) for t, w in ((q, blk.q_ln), (k, blk.k_ln)))
        for rows in torch.arange(len(ids)).split(lengths):
            if len(rows):
                heads = lambda t: t[rows].reshape(1, -1, H, 64).transpose(1, 2)  # noqa: E731
                ref = oe.attention(oe.rope(heads(q)), oe.rope(heads(k)), heads(v)).transpose(1, 2).reshape(len(rows), D)
                # fp16's roundings of q, k and p: 4e-4 of a value or so each way, independent, six times that at most
                assert float((o[rows] - ref).abs().max()) <= 1e-2 * float(ref.pow(2).mean().sqrt())
        a = product(at + 1, "wo")
        _check8(seen[at + 2][1], hs[i], a, alpha, blk.ln2_w, blk.ln2_b, "layer", 1e-5)
        product(at + 2, "w1", "silu")
        m = product(at + 3, "w2")
        mid = hs[i] + a.float() * alpha
        if i + 1 < len(model.layers):
            nxt = model.layers[i + 1]
            ref = mid.double() + alpha * m.double()
            # alpha, alpha a, its sum here and in the kernel, alpha m and the second sum: a rounding each, 2^-24 of themselves
            size = mid.abs() + hs[i + 1].abs() + alpha * (a.float().abs() + m.float().abs())
            assert bool(((hs[i + 1].double() - ref).abs() <= 2.0 ** -22 * size.double()).all())
            _check8(seen[at + 4][1], mid, m, alpha, nxt.ln1_w, nxt.ln1_b, "layer", 1e-5)
        else:
            ref = F.layer_norm(mid.double() + alpha * m.double(), (D,), model.norm_w.double(), None, 1e-5)
            assert float((hs[-1].double() - ref).abs().max()) <= 1e-4 * float(ref.pow(2).mean().sqrt())
    # the padded form takes the same linears, its rows through fp16 first: e4m3's error of both, no more
    a, b = model(input_ids=ids[None, :lengths[0]]).hidden_states[-1, 0], hs[-1, :lengths[0]]
    assert float((a - b).pow(2).mean().sqrt()) <= 0.15


def test_packed_rows_captured_and_what_takes_the_place_of_a_part(gpu_lib, pkg):
    hf = _hf(256, 384, 2, 5)
    model = pkg.esmc.HipEsmc.from_hf(hf, n_heads=4, linear=pkg.f8.F8Linear, fused=True)
    ids = torch.randint(0, 33, (150,), generator=_gen(3)).to(DEV)
    cu = i32(0, 100, 149, 150)
    want = model.packed_hidden_states(ids, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.packed_hidden_states(ids, cu)
    keep = pkg.scratch.current(DEV)
    for _ in range(3):
        got.zero_()
        graph.replay()
        again = model.packed_hidden_states(ids, cu)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, want)
    del keep
    blk, seen = model.layers[1], []
    blk.ffn = lambda h: seen.append(h.shape) or pkg.esmc.EsmcBlock.ffn(blk, h)
    assert not blk.takes_rows()
    other = model.packed_hidden_states(ids, cu)
    assert seen == [(150, 256)] and float((other[-1] - want[-1]).pow(2).mean().sqrt()) <= 0.15
    with pytest.raises(ValueError):
        pkg.esmc.HipEsmc.from_hf(hf, n_heads=4, fused=True)
    with pytest.raises(ValueError):
        pkg.esmc.EsmcBlock(*(getattr(blk, n) for n in pkg.esmc.NORMS), blk.wqkv, blk.wo,
                           pkg.f8.F8Linear.from_float(torch.zeros(2 * 320, 256), gated=True), blk.w2, 4)


def _rows8(pkg, x, y, w):
    s, h = pkg.kernels.add_norm_f8(x, y, w)
    rows = pkg.f8.F8Rows(*h, x.shape[:1], x.shape[1], y.dtype)
    return s, rows.codes.view(torch.uint8), rows.scales


def test_rows_of_a_cache_without_sequences_read_as_zeros(gpu_lib, pkg):
    cache = pkg.cache4.Cache4(2, 2, 64)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    for _ in range(2):  # (memory that held something else)
        torch.full((2, 900, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        for t in cache.read(i32(0), none, none.view(0, 3), rows=900):
            assert t.shape == (900, 2, 64) and not bool(t.any())


def _calls(pkg):
    """Each call's ordinary forms, results as lists of tensors."""
    k = pkg.kernels
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s, t=torch.bfloat16: torch.randn(*s, generator=g, device=DEV).to(t)  # noqa: E731
    for T, D in ((1, 640), (9, 2560), (300, 1104)):
        w, b = r(D, t=torch.float32), r(D, t=torch.float32)
        for x, y in ((r(T, D), r(T, D)), (r(T, 2 * D, t=torch.float32)[:, :D], r(T, D))):
            yield lambda x=x, y=y, w=w, b=b: k.add_norm(x, y, w, b, norm="layer", alpha=0.5)
            # (codes and scales of rows behind the last are left as they were: the rows as values)
            yield lambda x=x, y=y, w=w: _rows8(pkg, x, y, w)
    for M, K, N in ((1, 2560, 1024), (5, 5120, 640), (238, 2560, 640)):
        x, res = r(M, K), r(M, N)
        for gated in (False, True):
            lin = pkg.linear.Linear16.from_float(r(N, K), r(N), gated=gated, dtype=torch.bfloat16)
            e8 = pkg.f8.F8Linear.from_float(r(N, K), bias=r(N), gated=gated)
            rr = res[:, :N // 2].contiguous() if gated else res
            yield lambda lin=lin, x=x, rr=rr: (lin(x, "gelu", rr, 0.25),)
            rows = pkg.f8.F8Rows(*k.add_norm_f8(x, None)[1], (M,), K, torch.bfloat16)
            yield lambda e8=e8, rows=rows, rr=rr: (e8(rows, "silu", rr, 0.25),)
    for nq, nk in (([1, 1], [300, 5000]), ([40, 3], [64, 700])):
        case = Case(pkg, nq, nk, 8, 2, 64, torch.bfloat16)
        yield lambda c=case: (c.fill().cache.data.clone(), *c.cache.read(c.whole, c.lens, c.table))
        yield lambda c=case: (c.fill().attend(), c.attend(causal=False, scale=0.3))


def test_both_ways_give_the_same_bits(gpu_lib, pkg, monkeypatch):
    if pkg.capi.bind is pkg.capi._LongWay:
        pytest.skip("the native module could not be built here")
    calls = list(_calls(pkg))
    short = [f() for f in calls]
    with monkeypatch.context() as m:
        m.setattr(pkg.capi, "bind", pkg.capi._LongWay)
        longer = [f() for f in calls]
    for i, (a, b) in enumerate(zip(short, longer)):
        assert len(a) == len(b) and all(s.dtype is t.dtype and torch.equal(s, t) for s, t in zip(a, b)), i
    # a third time, on a stream of its own
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = [f() for f in calls]
    stream.synchronize()
    for i, (a, b) in enumerate(zip(short, other)):
        assert all(torch.equal(s, t) for s, t in zip(a, b)), i


def test_both_ways_refuse_the_same(gpu_lib, pkg, monkeypatch):
    k = pkg.kernels
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    lin = pkg.linear.Linear16.from_float(torch.zeros(64, 64), dtype=torch.bfloat16)
    case = Case(pkg, [1], [64], 4, 2, 64, torch.bfloat16)
    c = case.cache.data
    calls = [
        (lambda: k.add_norm(x, x[:, :32]), -2), (lambda: k.add_norm(x, x.half()), -4), (lambda: k.add_norm(x, x, x[0]), -2),
        (lambda: k.add_norm(x, x, eps=-1.0), -2), (lambda: k.add_norm(x, x, alpha=math.inf), -2), (lambda: k.add_norm(x, x, norm="max"), -4),
        (lambda: k.add_norm(x.cpu(), x), -5), (lambda: k.add_norm(x, x.expand(2, 4, 64)[0].t().contiguous().t()), -3),
        (lambda: k.linear16(x, lin.packed[:-1], 64), -2), (lambda: k.linear16(x, lin.packed, 64, x[0]), -2),
        (lambda: k.linear16(x, lin.packed, 64, activation="tanh"), -4), (lambda: k.linear16(x, lin.packed, 64, alpha=math.nan), -2),
        (lambda: k.linear16(x, lin.packed, 64, residual=x[:3]), -2), (lambda: k.linear16(x, lin.packed, 72), -2),
        (lambda: k.cache4_append(c, case.k, case.v[:, :1], case.whole, case.lens, case.table), -2),
        (lambda: k.cache4_append(c, case.k, case.v, case.whole, case.lens, case.table.long()), -2),
        (lambda: k.cache4_append(c[:-1], case.k, case.v, case.whole, case.lens, case.table), -2),
        (lambda: k.cache4_attention(c, case.q, 3, case.cu, case.lens, case.table), -2),
        (lambda: k.cache4_attention(c, case.q, 2, case.cu[:-1], case.lens, case.table), -2),
        (lambda: k.cache4_attention(c, case.q, 2, case.cu, case.lens, case.table, True, math.inf), -2),
        (lambda: k.cache4_attention(c, case.q.cpu(), 2, case.cu, case.lens, case.table), -5),
    ]

    def codes():
        found = []
        for f, _ in calls:
            with pytest.raises(pkg.capi.EsmError) as e:
                f()
            found.append(e.value.code)
        return found

    short = codes()
    monkeypatch.setattr(pkg.capi, "bind", pkg.capi._LongWay)
    assert short == codes() == [c for _, c in calls]


def test_nothing_to_do(gpu_lib, pkg):
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    x = torch.zeros(0, 256, dtype=torch.bfloat16, device=DEV)
    s, rows = pkg.norm.AddNorm(torch.ones(256))(x, x, f8=True)
    assert s.shape == (0, 256) and rows.dequantized().shape == (0, 256) and rows.codes.shape == (0, 256)
    w = torch.ones(128, 256, device=DEV)
    for gated in (False, True):
        lin, e8 = pkg.linear.Linear16.from_float(w, gated=gated, dtype=torch.bfloat16), pkg.f8.F8Linear.from_float(w, bias=w[:, 0], gated=gated)
        for y in (lin(x, "silu"), e8(x, "gelu"), e8(rows), lin(x.view(3, 0, 256))):
            assert y.shape[-1] == lin.out_features and not y.numel() and y.dtype is torch.bfloat16
    cache = pkg.cache4.Cache4(2, 2, 64)
    q, k = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    for cu, lens, table in ((i32(0), none, none.view(0, 2)), (i32(0, 0), i32(5), i32(0).view(1, 1)), (i32(0, 0), i32(0), none.view(1, 0))):
        cache.append(k, k, cu, lens, table)
        assert cache.attend(q, cu, lens, table).shape == (0, 4, 64) and not bool(cache.data.any())
        assert all(t.shape == (0, 2, 64) for t in cache.read(cu, lens, table))
    # queries of sequences without keys or without a table: zeros; a cache without pages holds nothing
    q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    empty = pkg.cache4.Cache4(0, 2, 64)
    for c, lens, table in ((cache, i32(0, 0), i32(0, 1).view(2, 1)), (cache, i32(70, 9), none.view(2, 0)), (empty, i32(7, 1), i32(0, 0).view(2, 1))):
        assert not bool(c.attend(q, i32(0, 2, 3), lens, table).any())
        c.append(q[:, :2].contiguous(), q[:, :2].contiguous(), i32(0, 2, 3), lens, table if c is empty else none.view(2, 0))
    assert not bool(cache.data.any())


def test_offsets_past_32_bits(gpu_lib, pkg):
    g = torch.Generator(device=DEV).manual_seed(5)
    dt, D, T = torch.bfloat16, 8192, 270_000  # rows of 4.4 GB
    x = torch.empty(T, D, dtype=dt, device=DEV)
    x[-40:] = torch.randn(40, D, generator=g, device=DEV).to(dt)
    x[:-40] = x[-1]
    w = torch.ones(D, device=DEV)
    s, h = pkg.kernels.add_norm(x, x, w)
    few = pkg.kernels.add_norm(x[-40:].clone(), x[-40:].clone(), w)
    # (few rows divide a row between more waves: sums in another order)
    assert torch.equal(s[-40:], few[0]) and float((h[-40:].float() - few[1].float()).abs().max()) <= 2.0 ** -7 * float(few[1].abs().max())
    assert torch.equal(h[0], h[-1]) and torch.equal(h[T // 2], h[-1])
    del s, h
    lin = pkg.linear.Linear16.from_float(torch.randn(D, 64, generator=g, device=DEV) / 8, dtype=dt)
    y = lin(x[:, :64])
    assert y.shape == (T, D)
    check_linear16(y[-40:], x[-40:, :64].contiguous(), lin.weight, None, None, False, None, 1.0)
    assert torch.equal(y[0], y[-1]) and torch.equal(y[T // 2], y[-1])
    del x, y
    # a cache of 4.5 GB: its first and last pages
    cache = pkg.cache4.Cache4(62_000, 8, 128, dtype=dt)
    table = i32(61_999, 1, 61_500, 30_000, 0).view(1, 5)
    k, v = (torch.randn(300, 8, 128, generator=g, device=DEV).to(dt) for _ in range(2))
    q = torch.randn(2, 16, 128, generator=g, device=DEV).to(dt)
    cache.append(k, v, i32(0, 300), i32(300), table)
    held = [C4.hold(t) for t in (k, v)]
    for got, (c, s, z) in zip(cache.read(i32(0, 300), i32(300), table), held):
        assert torch.equal(got, (s * (c - z)).to(dt))
    ref, bound = C4.attention(q, *held, True, 128 ** -0.5)
    assert bool(((cache.attend(q, i32(0, 2), i32(300), table).double() - ref).abs() <= bound).all())
