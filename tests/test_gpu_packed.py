"""Attention over packed sequences against a 64-bit restatement of its definition, with bounds from the arithmetic."""

import math
import threading

import pytest
import torch

from oracle import packed as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _case(nq, nk, H, Hk, d, dtype, seed=0, tail=0):
    """q, k, v as views of wider rows, with ``tail`` rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    if nk is None:
        T = sum(nq) + tail
        qkv = torch.randn(T, (H + 2 * Hk) * d, generator=g).to(dtype).to(DEV)
        q, k, v = qkv.split([H * d, Hk * d, Hk * d], dim=1)
        nk = nq
    else:
        q = torch.randn(sum(nq) + tail, H * d, generator=g).to(dtype).to(DEV)
        kv = torch.randn(sum(nk) + tail, 2 * Hk * d, generator=g).to(dtype).to(DEV)
        k, v = kv.split([Hk * d, Hk * d], dim=1)
    return (q.unflatten(1, (H, d)), k.unflatten(1, (Hk, d)), v.unflatten(1, (Hk, d)), _starts(nq), _starts(nk))


def _cu(c):
    return torch.tensor(c, dtype=torch.int32, device=DEV)


def _check(got, o, bound, what=""):
    got = got.detach().cpu().double()
    live = ~torch.isnan(bound) & ~torch.isnan(o)
    err = (got - o).abs()
    assert bool(torch.isfinite(got[live]).all()), what
    worst = (err / bound.clamp_min(1e-300))[live].max() if live.any() else torch.tensor(0.0)
    assert float(worst) <= 1.0, f"{what}: error {float(worst):.2f} of its bound"


SHAPES = [  # query heads, key heads, head size
    (2, 2, 64), (8, 2, 128), (4, 1, 80), (3, 3, 8), (6, 2, 40), (5, 1, 128), (64, 1, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,d", SHAPES)
def test_sequences_of_many_lengths(gpu_lib, pkg, H, Hk, d, causal, dtype):
    # one row, none, tile borders and beyond; six rows behind the last sequence are left as they were
    nq = [1, 0, 31, 33, 64, 65, 130, 7]
    q, k, v, cq, ck = _case(nq, None, H, Hk, d, dtype, seed=H + d, tail=6)
    out = torch.full((q.shape[0], H, d), 7.0, dtype=dtype, device=DEV)
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), causal=causal, out=out)
    assert got is out
    o, bound = O.attention(q, k, v, cq, ck, causal, d ** -0.5)
    _check(got, o, bound)
    assert bool((got[cq[-1]:] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64), (4, 1, 80)])
def test_single_tokens_against_caches(gpu_lib, pkg, H, Hk, d, dtype):
    # one new row each: caches of one key, around the passes, and of none (the row is 0)
    nk = [1, 0, 127, 128, 129, 700, 257, 2050]
    q, k, v, cq, ck = _case([1] * len(nk), nk, H, Hk, d, dtype, seed=d)
    for causal in (False, True):
        got = pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), causal=causal)
        o, bound = O.attention(q, k, v, cq, ck, causal, d ** -0.5)
        _check(got, o, bound)
        assert bool((got[1] == 0).all())


@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64)])
def test_queries_and_keys_of_different_lengths(gpu_lib, pkg, H, Hk, d):
    # continued prompts; the last has more queries than keys: causal, its first rows see nothing and are 0
    nq, nk = [5, 40, 1, 90, 20], [300, 40, 66, 333, 12]
    q, k, v, cq, ck = _case(nq, nk, H, Hk, d, torch.bfloat16, seed=3)
    for causal in (False, True):
        got = pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), causal=causal, scale=0.2)
        o, bound = O.attention(q, k, v, cq, ck, causal, 0.2)
        _check(got, o, bound)
    assert bool((got[cq[4]:cq[4] + 8] == 0).all()) and bool((got[cq[4] + 8] != 0).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,d,causal", [(40, 40, 64, False), (32, 8, 128, True), (20, 4, 80, True)])
def test_many_rows(gpu_lib, pkg, H, Hk, d, causal, dtype):
    # enough rows for the tiles that share their keys; a few heads are compared (the oracle is slow)
    nq = [513, 700, 1, 255, 256]
    q, k, v, cq, ck = _case(nq, None, H, Hk, d, dtype, seed=5)
    q[-256:] *= 6  # strong scores: the running maximum moves
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), causal=causal)
    G = H // Hk
    for hk in {0, Hk - 1}:
        hs = slice(hk * G, hk * G + 1)
        o, bound = O.attention(q[:, hs], k[:, hk:hk + 1], v[:, hk:hk + 1], cq, ck, causal, d ** -0.5)
        _check(got[:, hs], o, bound, f"key head {hk}")


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_unseen_rows_hold_reaches_nothing(gpu_lib, pkg, dtype, many):
    # later keys and values of infinities and NaN: rows that do not see them are finite, those that do follow the
    # formula; other sequences' rows and the rows behind the last sequence never count
    H, Hk, d = (40, 40, 64) if many else (4, 2, 128)
    nq = [300, 420, 65] if many else [70, 33, 65]
    q, k, v, cq, ck = _case(nq, None, H, Hk, d, dtype, seed=9, tail=40)
    bad = torch.tensor([math.inf, -math.inf, math.nan, math.inf], dtype=dtype, device=DEV)
    at = cq[1] + 20
    v[at, 0, :4] = bad                      # seen by the rows from 20 on of the second sequence
    v[cq[2] + 64, 0] = math.nan             # by the last row of the third alone
    k[cq[2] + 50, 1, 3] = math.nan          # by the rows from 50 on
    v[at + 5, 0, 0] = -math.inf             # +inf from row 20, NaN with -inf from row 25 on
    for t in (q, k, v):
        t[cq[-1]:] = math.nan
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), causal=True).float().cpu()
    clean = [t.clone() for t in (k, v)]
    clean[0][cq[2] + 50, 1, 3] = 0
    clean[1][at, 0, :4] = clean[1][at + 5, 0, 0] = clean[1][cq[2] + 64, 0] = 0
    G = H // Hk
    for h in (0, G):
        o, bound = O.attention(q[:cq[-1], h:h + 1], *(t[:cq[-1], h // G:h // G + 1] for t in clean), cq, ck, True, d ** -0.5)
        rows = [i for i in range(cq[-1]) if not (cq[1] + 20 <= i < cq[2] or i == cq[2] + 64 or i >= cq[2] + 50)]
        _check(got[rows][:, h:h + 1], o[rows], bound[rows])
        if h == 0:
            cols = list(range(4, d))        # the rows that see the four odd values: every other column
            late = list(range(cq[1] + 26, cq[2]))
            _check(got[late][:, h:h + 1, cols], o[late][..., cols], bound[late][..., cols])
    s = got[at:at + 5, 0]
    assert bool((s[:, 0] == math.inf).all() and (s[:, 1] == -math.inf).all() and s[:, 2].isnan().all())
    assert bool((s[:, 3] == math.inf).all()) and bool(got[at + 5:cq[2], 0, 0].isnan().all())
    assert bool(got[cq[2] + 64, 0].isnan().all())
    assert bool(got[cq[2] + 50:cq[3], G].isnan().all())


@pytest.mark.parametrize("decode", [False, True])
def test_more_sequences_than_a_wave(gpu_lib, pkg, decode):
    g = torch.Generator().manual_seed(1)
    n = 150
    nq = [1] * n if decode else torch.randint(0, 40, (n,), generator=g).tolist()
    nk = torch.randint(0, 300, (n,), generator=g).tolist() if decode else None
    q, k, v, cq, ck = _case(nq, nk, 4, 2, 64, torch.float16, seed=2, tail=3)
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), causal=True)
    o, bound = O.attention(q, k, v, cq, ck, True, 0.125)
    _check(got, o, bound)


def test_sequences_of_one_length_and_of_many_levels(gpu_lib, pkg):
    # the order that takes the longest tiles first must visit each tile once: equal lengths, and lengths that differ by
    # every level, with and without cached keys
    for nq, nk in (([256] * 9, None), ([16 * i for i in range(1, 33)], None), ([200] * 6, [200 + 300 * i for i in range(6)]),
                   ([700, 1], [700, 5000])):
        q, k, v, cq, ck = _case(nq, nk, 16, 2, 64, torch.bfloat16, seed=len(nq))
        for causal in (False, True):
            out = torch.full_like(q, math.nan, memory_format=torch.contiguous_format)
            pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), causal=causal, out=out)
            o, bound = O.attention(q[:, 9:10], k[:, 1:], v[:, 1:], cq, ck, causal, 0.125)
            _check(out[:, 9:10], o, bound)
            assert bool(torch.isfinite(out).all())


def test_offsets_past_32_bits(gpu_lib, pkg):
    # a cache of 9.4 GB whose last sequences lie beyond 2^32 bytes (and 2^31 elements)
    rows, Hk, d = 2300000, 8, 128
    kv = torch.empty(rows, 2 * Hk * d, dtype=torch.bfloat16, device=DEV)
    nk = [300, 77]
    kv[-sum(nk):] = torch.randn(sum(nk), 2 * Hk * d, generator=torch.Generator().manual_seed(0)).to(DEV)
    k, v = (t.unflatten(1, (Hk, d)) for t in kv.split([Hk * d, Hk * d], dim=1))
    q = torch.randn(130, 16, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    first = rows - sum(nk)
    for nq in ([1, 1], [128, 2], [100, 30]):
        cq, ck = _starts(nq), [first, first + 300, rows]
        got = pkg.kernels.packed_attention(q[:cq[-1]], k, v, _cu(cq), _cu(ck), causal=True)
        o, bound = O.attention(q[:cq[-1], 2:3], k[first:, 1:2], v[first:, 1:2], cq, [0, 300, 377], True, d ** -0.5)
        _check(got[:, 2:3], o, bound)


def test_large_scores_and_equal_ones(gpu_lib, pkg):
    # scores of several thousands, where only the maximum survives, and all equal ones, whose mean is exact to bounds
    q, k, v, cq, ck = _case([90, 40], None, 2, 2, 64, torch.bfloat16, seed=4)
    q[:90] *= 300
    q[90:] = 0
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq))
    o, bound = O.attention(q, k, v, cq, ck, False, 0.125)
    _check(got, o, bound)


def test_starts_outside_the_rows_are_brought_inside(gpu_lib, pkg):
    q, k, v, cq, _ = _case([40, 30], None, 2, 1, 64, torch.float16, seed=2)
    good = pkg.kernels.packed_attention(q, k, v, _cu([0, 40, 70]))
    wild = pkg.kernels.packed_attention(q, k, v, _cu([-5, 40, 1000000]))
    assert torch.equal(good, wild)
    kept = torch.full_like(good, 3.0)  # falling starts: a sequence without rows
    pkg.kernels.packed_attention(q, k, v, _cu([70, 20, 10]), out=kept)
    assert bool((kept == 3.0).all())


def test_layouts_and_in_place(gpu_lib, pkg):
    # heads outside rows, a strided output, the output over the queries: the same bits
    q, k, v, cq, _ = _case([100, 61], None, 4, 2, 64, torch.bfloat16, seed=6)
    cu = _cu(cq)
    ref = pkg.kernels.packed_attention(q, k, v, cu, causal=True)
    t = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    assert torch.equal(ref, pkg.kernels.packed_attention(t(q), t(k), t(v), cu, causal=True))
    wide = torch.zeros(161, 4, 96, dtype=torch.bfloat16, device=DEV)
    pkg.kernels.packed_attention(q, k, v, cu, causal=True, out=wide[..., 16:80])
    assert torch.equal(ref, wide[..., 16:80]) and bool((wide[..., :16] == 0).all() and (wide[..., 80:] == 0).all())
    qc = q.contiguous()
    assert torch.equal(ref, pkg.kernels.packed_attention(qc, k, v, cu, causal=True, out=qc))


def test_empty_calls(gpu_lib, pkg):
    e = lambda *s: torch.empty(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    assert pkg.kernels.packed_attention(e(0, 2, 64), e(0, 2, 64), e(0, 2, 64), _cu([0])).shape == (0, 2, 64)
    assert pkg.kernels.packed_attention(e(0, 2, 64), e(0, 2, 64), e(0, 2, 64), _cu([0, 0, 0])).shape == (0, 2, 64)
    got = pkg.kernels.packed_attention(e(5, 2, 64).zero_(), e(0, 2, 64), e(0, 2, 64), _cu([0, 5]), _cu([0, 0]))
    assert bool((got == 0).all())


@pytest.mark.parametrize("nq,nk", [([300, 20], None), ([1] * 6, [900, 3, 2000, 65, 0, 128])])
def test_graph_and_side_stream(gpu_lib, pkg, nq, nk):
    q, k, v, cq, ck = _case(nq, nk, 8, 2, 128, torch.bfloat16, seed=8)
    cuq, cuk = _cu(cq), _cu(ck)
    ref = pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ref, other)
    out = torch.empty_like(ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True, out=out)
    keep = pkg.scratch.current(DEV)
    for _ in range(3):
        out.fill_(5.0)
        graph.replay()
        again = pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(again, ref)
    del keep


def test_two_threads_on_their_own_streams(gpu_lib, pkg):
    # calls whose chunks of keys meet in the device's one scratch buffer, beside linears that use it too
    q, k, v, cq, ck = _case([1] * 4, [5000, 70, 0, 2500], 8, 2, 128, torch.float16, seed=3)
    cuq, cuk = _cu(cq), _cu(ck)
    x = torch.randn(100, 640, generator=torch.Generator().manual_seed(0)).half().to(DEV)
    lin = pkg.f8.F8Linear.from_float(torch.randn(2560, 640, generator=torch.Generator().manual_seed(1)))
    ref, lref = pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True), lin(x)
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    a = pkg.kernels.packed_attention(q, k, v, cuq, cuk, causal=True)
                    b = lin(x)
                    if not (torch.equal(a, ref) and torch.equal(b, lref)):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001  (shown by the assertion)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_graphs_have_workspaces_of_their_own(gpu_lib, pkg):
    # two graphs whose rows have several chunks of keys, replayed at once, after the shared scratch has been given up
    cases, graphs, outs, refs = [], [], [], []
    for seed in (1, 2):
        q, k, v, cq, ck = _case([1] * 8, [6000, 900, 3, 2000, 65, 0, 128, 4100], 8, 2, 128, torch.bfloat16, seed=seed)
        cases.append((q, k, v, _cu(cq), _cu(ck)))
        refs.append(pkg.kernels.packed_attention(*cases[-1], causal=True))
    assert pkg.capi.lib().packed_attention_workspace_bytes(8, 8, cases[0][1].shape[0], 8, 2, 128) > 0
    before = pkg.scratch.generation(DEV)
    for c in cases:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pkg.kernels.packed_attention(*c, causal=True))
        graphs.append(graph)
    assert pkg.scratch.generation(DEV) == before
    with pkg.scratch.guard(DEV):
        pkg.scratch.get(pkg.scratch.current(DEV).numel() + 1, DEV).fill_(255)
    other = torch.full((1 << 22,), float("nan"), device=DEV)
    side = torch.cuda.Stream()
    for _ in range(5):
        for o in outs:
            o.fill_(7.0)
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(10):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    assert bool(other.isnan().all())


def test_refusals(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    x = torch.zeros(8, 4, 64, dtype=torch.float16, device=DEV)
    cu = _cu([0, 8])

    def refused(code, *a, **kw):
        with pytest.raises(E) as e:
            K.packed_attention(*a, **kw)
        assert e.value.code == code, str(e.value)

    refused(-2, x.float(), x, x, cu)
    refused(-2, x, x.bfloat16(), x, cu)
    refused(-2, x, x[:, :3], x[:, :3], cu)          # 4 heads in groups of 3 key heads
    refused(-2, x, x, x[:, :2], cu)
    refused(-2, x, x[:5], x[:5], cu)                # other rows without cu_k
    refused(-2, x, x, x, cu.long())
    refused(-2, x, x, x, cu, _cu([0, 4, 8]))
    refused(-5, x, x, x, cu.cpu())
    refused(-5, x.cpu(), x, x, cu)
    refused(-3, x[..., ::2], x[..., ::2], x[..., ::2], cu)
    refused(-3, x[..., 4:12], x[..., 4:12], x[..., 4:12], cu)      # not 16-byte aligned
    refused(-3, x[:1].expand(8, 4, 64), x, x, cu, out=x[:1].expand(8, 4, 64))
    refused(-3, x, x[:1].expand(8, 4, 64), x, cu)
    refused(-4, x[..., :60].contiguous(), x[..., :60].contiguous(), x[..., :60].contiguous(), cu)
    w = torch.zeros(8, 1, 136, dtype=torch.float16, device=DEV)
    refused(-4, w, w, w, cu)
    for s in (0.0, -1.0, math.nan, math.inf):
        refused(-2, x, x, x, cu, scale=s)
    refused(-2, x, x, x, cu, out=torch.zeros(8, 4, 32, dtype=torch.float16, device=DEV))
    refused(-3, x, x, x, cu, out=torch.zeros(8, 1, 64, dtype=torch.float16, device=DEV).expand(8, 4, 64))
    y = torch.zeros_like(x)
    refused(-3, x, y, x, cu, out=y)
    refused(-3, x, x.clone(), y, cu, out=y)
    buf = torch.zeros(8, 4, 64, dtype=torch.float16, device=DEV)
    refused(-3, buf[:, :2], x[:, :2], x[:, :2], cu, out=buf.view(-1)[:1024].view(8, 2, 64))  # over q, other strides
