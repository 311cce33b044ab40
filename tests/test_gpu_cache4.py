"""Keys and values in 4 bits and the attention on them, against 64 bits."""

import math
import threading

import pytest
import torch

from oracle import cache4 as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


class Case:
    """Sequences of nk keys in pages that lie anywhere, nq of them queries (the last ones if causal)."""

    def __init__(self, pkg, nq, nk, H, Hk, d, dtype, seed=0, spare=2):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
        pages = [-(-n // 64) for n in nk]
        where = torch.randperm(sum(pages) + spare, generator=g, device=DEV).int()
        self.table = torch.full((len(nk), max(pages) + 2), -1, dtype=torch.int32, device=DEV)  # (behind the last: no page)
        for i, (a, n) in enumerate(zip(_starts(pages), pages)):
            self.table[i, :n] = where[a:a + n]
        self.nq, self.nk, self.cq, self.ck = nq, nk, _starts(nq), _starts(nk)
        self.k, self.v = (r(self.ck[-1], Hk, d) + 0.5 * r(Hk, d)).to(dtype), r(self.ck[-1], Hk, d).to(dtype)
        self.q = (1.5 * r(self.cq[-1], H, d)).to(dtype)
        self.cu, self.lens = i32(*self.cq), i32(*nk)
        self.cache = pkg.cache4.Cache4(sum(pages) + spare, Hk, d, dtype=dtype)
        self.whole = i32(*self.ck)

    def fill(self):
        self.cache.append(self.k, self.v, self.whole, self.lens, self.table)
        return self

    def attend(self, **kw):
        return self.cache.attend(self.q, self.cu, self.lens, self.table, **kw)

    def check(self, o, causal=True, scale=None, keep=None):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        held = [O.hold(t) for t in (self.k, self.v)]
        for i, (nq, nk) in enumerate(zip(self.nq, self.nk)):
            if not nq:
                continue
            rows, keys = slice(self.cq[i], self.cq[i + 1]), slice(self.ck[i], self.ck[i + 1])
            ref, bound = O.attention(self.q[rows], *([t[keys] for t in h] for h in held), causal, scale, None if keep is None else keep[keys])
            got = o[rows].double()
            assert torch.equal(got.isnan(), ref.isnan()), i
            worst = float(torch.where(ref.isnan(), torch.zeros_like(ref), (got - ref).abs() / bound).max())
            assert worst <= 1.0, f"sequence {i}: error {worst:.2f} of its bound"


@pytest.mark.parametrize("d", [8, 64, 72, 80, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_written_and_read_back(gpu_lib, pkg, d, dtype):
    for Hk in (1, 3, 8, 40):
        c = Case(pkg, [1], [70, 1, 64, 200], Hk, Hk, d, dtype, seed=Hk)
        c.k[3, 0, :4] *= 1000  # a group with a range of its own
        c.k[5] = 0
        c.v[6] = 3.5
        c.v[7] = c.v[7] * 1e-3 + 7
        c.fill()
        for got, x in zip(c.cache.read(c.whole, c.lens, c.table), (c.k, c.v)):
            code, s, z = O.hold(x)
            assert torch.equal(got, (s * (code - z)).to(dtype))
            worst = float(((got.double() - x.double()).abs() - (0.5 + 2.0 ** -10) * s - 2 ** -8 * x.double().abs()).max())
            assert worst <= 0  # half a step, and a rounding


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_at_a_time_as_a_batch(gpu_lib, pkg, dtype):
    c = Case(pkg, [1, 1], [130, 33], 4, 2, 80, dtype).fill()
    other = Case(pkg, [1, 1], [130, 33], 4, 2, 80, dtype)
    n = [0, 0]
    while n != [130, 33]:  # tokens and small pieces, both sequences in a call
        step = [min(a, b - m) for a, b, m in zip((3, 1), (130, 33), n)]
        rows = torch.cat([torch.arange(other.ck[i] + n[i], other.ck[i] + n[i] + step[i]) for i in (0, 1)]).to(DEV)
        n = [a + b for a, b in zip(n, step)]
        other.cache.append(other.k[rows], other.v[rows], i32(0, step[0], sum(step)), i32(*n), other.table)
    assert torch.equal(c.cache.data, other.cache.data)


def test_only_the_rows_places_are_written(gpu_lib, pkg):
    for Hk, d in ((3, 72), (8, 128)):
        c = Case(pkg, [1], [300, 90], Hk, Hk, d, torch.bfloat16).fill()
        before = [t.clone() for t in c.cache.read(c.whole, c.lens, c.table)]
        spare = c.cache.data.view(c.cache.pages, -1)[[p for p in range(c.cache.pages) if p not in set(c.table.flatten().tolist())]]
        assert bool((spare == 0).all())
        # rows 100 .. 139 of the first again, with other values; rows of no sequence behind them; a length past the table, a bad page
        k = torch.randn(50, Hk, d, device=DEV).bfloat16()
        c.cache.append(k, k, i32(0, 40, 40), i32(140, 90), c.table)
        table = c.table.clone()
        table[0, 1] = c.cache.pages
        c.cache.append(k, k, i32(0, 30, 40), i32(100, 64 * table.shape[1] + 20), table)  # all of it without a place
        c.cache.append(k, k, i32(0, 10, 50), i32(4, -5), c.table)  # the first 6 stand before the first place
        after = c.cache.read(c.whole, c.lens, c.table)
        h = (lambda t: t[1] * (t[0] - t[2]))(O.hold(k)).bfloat16()
        for a, b in zip(before, after):
            a[100:140] = h[:40]
            a[0:4] = h[6:10]
            assert torch.equal(a, b)
        got = c.cache.read(i32(0, 10, 20), i32(4, 64 * c.table.shape[1] + 5), c.table, rows=25)
        assert bool((got[0][:6] == 0).all() and (got[0][10:] == 0).all()) and torch.equal(got[0][6:10], h[6:10])


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_with_nan_and_infinities(gpu_lib, pkg, dtype):
    c = Case(pkg, [1, 1], [80, 80], 2, 2, 128, dtype)
    c.k[3, 0, 70], c.k[90, 1, 0], c.v[10, 1, 5], c.v[100, 0, 127] = float("nan"), float("inf"), float("-inf"), float("nan")
    c.fill()
    rk, rv = c.cache.read(c.whole, c.lens, c.table)
    for got, x in ((rk, c.k), (rv, c.v)):
        bad = (~torch.isfinite(x.view(*x.shape[:2], 2, 64))).any(-1).repeat_interleave(64, -1)
        assert torch.equal(got.isnan(), bad)
    c.check(c.attend())


SHAPES = [([1], [1]), ([1, 1, 1, 1], [64, 65, 200, 31]), ([5, 0, 17], [5, 3, 600]), ([40], [40]), ([70, 3], [500, 1]), ([1, 1], [5000, 3]),
          ([9], [0]), ([30, 2], [10, 700]), ([3, 3, 3], [1000, 64, 128]), ([200], [900])]


@pytest.mark.parametrize("H,Hk,d", [(4, 4, 64), (8, 2, 128), (6, 2, 80), (3, 1, 8), (16, 1, 72), (20, 4, 120)])
@pytest.mark.parametrize("dtype", TYPES)
def test_against_the_definition(gpu_lib, pkg, H, Hk, d, dtype):
    for i, (nq, nk) in enumerate(SHAPES):
        c = Case(pkg, nq, nk, H, Hk, d, dtype, seed=i).fill()
        c.check(c.attend())
        c.check(c.attend(causal=False, scale=0.3), causal=False, scale=0.3)


def test_many_sequences(gpu_lib, pkg):
    nk = [1 + (37 * i) % 400 for i in range(150)]
    nq = [min(n, 1 + i % 3) for i, n in enumerate(nk)]
    c = Case(pkg, nq, nk, 8, 2, 64, torch.bfloat16).fill()
    c.check(c.attend())
    nk = [700 if i == 130 else 0 for i in range(150)]
    c = Case(pkg, [2 if i in (3, 130) else 0 for i in range(150)], nk, 8, 2, 64, torch.bfloat16).fill()
    o = c.attend()
    c.check(o)
    assert bool((o[:2] == 0).all())


def test_one_long_among_short(gpu_lib, pkg):
    c = Case(pkg, [1] * 9, [20000] + [30] * 8, 8, 2, 128, torch.float16).fill()
    c.check(c.attend())


@pytest.mark.parametrize("longest", [1500, 3000])  # with a tile a sequence for every CU: whole, and divided
def test_many_sequences_and_some_long(gpu_lib, pkg, longest):
    nk = [longest if i in (7, 140) else (i * 53) % 300 for i in range(150)]
    nq = [min(n, i % 3) for i, n in enumerate(nk)]
    c = Case(pkg, nq, nk, 8, 2, 64, torch.bfloat16).fill()
    c.check(c.attend())
    # a page of no cache in the middle of a divided sequence: its keys are not seen
    c.table[140, 11] = -7
    c.table[7, 3] = 1 << 30
    keep = torch.ones(c.ck[-1], dtype=torch.bool, device=DEV)
    keep[c.ck[140] + 704:c.ck[140] + 768] = False
    keep[c.ck[7] + 192:c.ck[7] + 256] = False
    c.check(c.attend(), keep=keep)


def test_pages_of_no_cache_and_shared_pages(gpu_lib, pkg):
    c = Case(pkg, [4, 4], [400, 400], 8, 2, 128, torch.bfloat16).fill()
    keep = torch.ones(800, dtype=torch.bool, device=DEV)
    for seq, page, bad in ((0, 2, -1), (0, 6, c.cache.pages), (1, 0, 2 ** 31 - 1), (1, 5, -2 ** 31)):
        c.table[seq, page] = bad
        keep[400 * seq + 64 * page:400 * seq + min(400, 64 * page + 64)] = False
    for causal in (True, False):
        c.check(c.attend(causal=causal), causal, keep=keep)
    c.table[:] = -1
    assert bool((c.attend() == 0).all())
    # two sequences that read the same pages
    c = Case(pkg, [2], [300], 8, 2, 128, torch.bfloat16).fill()
    o = c.attend()
    two = c.cache.attend(torch.cat([c.q, c.q]), i32(0, 2, 4), c.lens.repeat(2), c.table.repeat(2, 1))
    assert torch.equal(two[:2], o) and torch.equal(two[2:], o)


@pytest.mark.parametrize("nq", [1, 7, 60])
def test_what_unseen_places_hold_reaches_nothing(gpu_lib, pkg, nq):
    c = Case(pkg, [nq], [100], 8, 2, 128, torch.bfloat16).fill()
    want = c.attend()
    bad = torch.full((28, 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    c.cache.append(bad, bad, i32(0, 28), i32(128), c.table)  # behind the keys, in their last page
    assert torch.equal(c.attend(), want)
    if nq > 1:  # a later key that only the last row sees
        c.cache.append(bad[:1], bad[:1], i32(0, 1), c.lens, c.table)
        o = c.attend()
        assert torch.equal(o[:-1], want[:-1]) and bool(o[-1].isnan().all())


def test_rows_of_no_sequence_and_bad_starts(gpu_lib, pkg):
    c = Case(pkg, [3, 2], [90, 300], 8, 2, 80, torch.float16).fill()
    out = torch.full((9, 8, 80), 5.0, dtype=torch.float16, device=DEV)
    q = torch.cat([c.q, c.q[:4]])
    o = c.cache.attend(q, c.cu, c.lens, c.table, out=out)
    assert o is out and bool((o[5:] == 5).all()) and torch.equal(o[:5], c.attend())
    # lengths and starts outside what there is are brought inside: nothing to compare, nothing out of place
    for cu, lens in ((i32(-7, 3, 2 ** 30), i32(90, 300)), (i32(0, 3, 5), i32(-1, 2 ** 31 - 1)), (i32(5, 0, 5), i32(90, 300)), (i32(5, 5, 5), i32(9, 9))):
        y = c.cache.attend(c.q, cu, lens, c.table)
        c.cache.append(c.k[:5], c.v[:5], cu, i32(0, 0), c.table)
        c.cache.read(cu, lens, c.table, rows=5)
        assert y.shape == c.q.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_and_steps_of_every_size(gpu_lib, pkg, dtype):
    for scale_q, scale_k, scale_v in ((30, 1, 1), (1, 1e-4, 1e-4), (0.01, 100, 200), (200, 30, 1)):
        c = Case(pkg, [2, 1], [300, 700], 4, 2, 64, dtype)
        c.q, c.k, c.v = c.q * scale_q, c.k * scale_k, c.v * scale_v
        c.fill()
        c.check(c.attend())
    if dtype is torch.bfloat16:  # values beyond fp16's
        c = Case(pkg, [2], [300], 4, 2, 64, dtype)
        c.v, c.k, c.q = c.v * 1e20, c.k * 1e10, c.q * 1e-10
        c.fill()
        c.check(c.attend())
    # values with steps far apart along the keys
    c = Case(pkg, [1], [500], 4, 2, 128, dtype)
    c.v *= torch.logspace(-3, 3, 500, device=DEV)[:, None, None].to(dtype)
    c.fill()
    c.check(c.attend())


def test_views_and_out(gpu_lib, pkg):
    c = Case(pkg, [5, 60], [200, 100], 8, 2, 64, torch.bfloat16).fill()
    want = c.attend()
    wide = torch.full((65, 12, 72), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 2:10, :64] = c.q
    assert torch.equal(c.cache.attend(wide[:, 2:10, :64], c.cu, c.lens, c.table), want)
    kv = torch.full((300, 6, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    kv[:, 1:3], kv[:, 4:6] = c.k, c.v
    other = pkg.cache4.Cache4(c.cache.pages, 2, 64, dtype=torch.bfloat16)
    other.append(kv[:, 1:3], kv[:, 4:6], c.whole, c.lens, c.table)
    assert torch.equal(other.data, c.cache.data)
    q = c.q.clone()
    assert c.cache.attend(q, c.cu, c.lens, c.table, out=q) is q and torch.equal(q, want)
    again = [c.attend() for _ in range(3)]
    assert all(torch.equal(a, want) for a in again)  # the same bits


@pytest.mark.parametrize("rows", [1, 4])
def test_steps_captured_and_replayed_with_growing_lengths(gpu_lib, pkg, rows):
    c = Case(pkg, [rows] * 3, [3000, 700, 40], 8, 2, 128, torch.bfloat16)
    n = [2500, 300, 4]
    for i in range(3):
        a = c.ck[i]
        c.cache.append(c.k[a:a + n[i]], c.v[a:a + n[i]], i32(0, n[i]), i32(n[i]), c.table[i:i + 1])
    q, k, v = c.q.clone(), c.k[:3 * rows].clone(), c.v[:3 * rows].clone()
    lens = i32(*n)

    def step():
        lens.add_(rows)
        c.cache.append(k, v, c.cu, lens, c.table)
        return c.cache.attend(q, c.cu, lens, c.table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.cache.attend(q, c.cu, lens, c.table)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    pkg.scratch.release()  # (the graph's workspace is its own)
    for turn in range(9):
        at = [m + turn * rows for m in n]
        idx = torch.cat([torch.arange(c.ck[i] + at[i], c.ck[i] + at[i] + rows) for i in range(3)]).to(DEV)
        k.copy_(c.k[idx]), v.copy_(c.v[idx])
        q.normal_()
        graph.replay()
        assert torch.equal(out, c.cache.attend(q, c.cu, lens, c.table))
        held = [O.hold(t) for t in (c.k, c.v)]
        for i in range(3):
            keys = slice(c.ck[i], c.ck[i] + at[i] + rows)
            ref, bound = O.attention(q[rows * i:rows * (i + 1)], *([t[keys] for t in h] for h in held), True, 128 ** -0.5)
            assert float(((out[rows * i:rows * (i + 1)].double() - ref).abs() / bound).max()) <= 1.0


def test_two_threads_on_their_own_streams(gpu_lib, pkg):
    cases = [Case(pkg, [1] * 4, [5000, 100, 900, 3000], 8, 2, 128, torch.bfloat16, seed=s).fill() for s in (0, 1)]
    want = [c.attend() for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(15):
                o = cases[i].attend()
                torch.cuda.current_stream().synchronize()
                if not torch.equal(o, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals(gpu_lib, pkg):
    E = pkg.capi.EsmError
    K = pkg.kernels
    c = Case(pkg, [2, 1], [90, 5], 8, 2, 64, torch.bfloat16).fill()
    q, at, data = c.q, (c.cu, c.lens, c.table), c.cache.data
    for code, call in ((-5, lambda: K.cache4_attention(data, q.cpu(), 2, *at)), (-5, lambda: K.cache4_attention(data.cpu(), q, 2, *at)),
                       (-5, lambda: K.cache4_attention(data, q, 2, c.cu.cpu(), c.lens, c.table)), (-2, lambda: K.cache4_attention(data, q, 3, *at)),
                       (-2, lambda: K.cache4_attention(data, q, 0, *at)), (-2, lambda: K.cache4_attention(data, q.float(), 2, *at)),
                       (-2, lambda: K.cache4_attention(data, q, 2, c.cu[:2], c.lens, c.table)), (-2, lambda: K.cache4_attention(data, q, 2, c.cu, c.lens, c.table[:1])),
                       (-2, lambda: K.cache4_attention(data, q, 2, c.cu.long(), c.lens, c.table)), (-3, lambda: K.cache4_attention(data, q, 2, c.cu, c.lens, c.table[:, ::2])),
                       (-2, lambda: K.cache4_attention(data[:-16], q, 2, *at)), (-2, lambda: K.cache4_attention(data, q, 2, *at, scale=0.0)),
                       (-2, lambda: K.cache4_attention(data, q, 2, *at, scale=float("nan"))), (-3, lambda: K.cache4_attention(data, q, 2, *at, out=q[:1].expand(3, 8, 64))),
                       (-2, lambda: K.cache4_append(data, c.k, c.v[:3], *at)), (-2, lambda: K.cache4_append(data, c.k.float(), c.v, *at)),
                       (-3, lambda: K.cache4_append(data, c.k.transpose(1, 2).contiguous().transpose(1, 2), c.v, *at)),
                       (-2, lambda: K.cache4_read(data, 3, 2, 64, torch.float32, *at))):
        with pytest.raises(E) as e:
            call()
        assert e.value.code == code, e.value
    for bad in (dict(heads=0), dict(head_dim=136), dict(head_dim=60), dict(pages=-1), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            pkg.cache4.Cache4(**{**dict(pages=2, heads=2, head_dim=64), **bad})
    for call in (lambda: c.cache.append(c.k.half(), c.v.half(), *at), lambda: c.cache.append(c.k[:, :1], c.v, *at), lambda: c.cache.attend(q[..., :56], *at),
                 lambda: c.cache.attend(q.half(), *at)):
        with pytest.raises(ValueError):
            call()
    none = pkg.cache4.Cache4(0, 2, 64)
    assert bool((none.attend(q, c.cu, c.lens, c.table) == 0).all())
    none.append(c.k[:3], c.v[:3], c.cu, c.lens, c.table)
    assert c.cache.attend(q[:0], i32(0), i32(), c.table[:0]).shape == (0, 8, 64) and c.cache.read(i32(0), i32(), c.table[:0])[0].shape == (0, 2, 64)
    assert math.isclose(c.cache.data.numel(), c.cache.pages * 2 * 64 * (64 + 8))
