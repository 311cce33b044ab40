"""Packed attention where sequences, scores and probabilities reach their ends: no keys at all, scores of -inf and of the
type's lowest value, scores of any size and probabilities far below their row's largest, against the formula."""

import math

import pytest
import torch

from oracle import packed as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _cu(c):
    return torch.tensor(c, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows", [[16], [40, 0, 300], [2000], [3] * 70])
def test_rows_without_any_keys_are_zero(gpu_lib, pkg, rows, causal, dtype):
    # no sequence has a key: every row sees none, whichever kernel the rows' number selects; the last row is of no sequence
    H, Hk, d, T = 8, 2, 64, sum(rows)
    q = torch.randn(T + 1, H, d, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    k = v = torch.empty(0, Hk, d, dtype=dtype, device=DEV)
    cq = [0]
    for n in rows:
        cq.append(cq[-1] + n)
    out = torch.full_like(q, 7.0)
    pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu([0] * len(cq)), causal=causal, out=out)
    assert bool((out[:T] == 0).all()) and bool((out[T:] == 7.0).all())


# ---- seen keys whose score is -inf, or the least a score can be ------------------------------------------


def _masked(nq, nk, bad, H, Hk, d, dtype, low, seed=0):
    """q, k, v whose scores at the keys ``bad`` of every sequence are ``low`` (a mask carried in the last value of a
    head: 1 in every query, ``low`` in those keys and 0 in the others) and which of each sequence's keys are left."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(nq), H, d, generator=g).to(dtype)
    k, v = (torch.randn(sum(nk), Hk, d, generator=g).to(dtype) for _ in range(2))
    q[..., -1], k[..., -1] = 1, 0
    at, left = 0, []
    for n in nk:
        gone = sorted(i for i in bad if i < n)
        k[[at + i for i in gone], :, -1] = low
        left.append([i for i in range(n) if i not in set(gone)])
        at += n
    return q.to(DEV), k.to(DEV), v.to(DEV), left


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _check_without(pkg, q, k, v, nq, nk, left, causal, scale, heads, what=""):
    """The kernel on all keys against the oracle on those that are left (a key of no weight is as none: with the
    masked keys before every other, or before every query's last, the causal limit stays where it is)."""
    cq, ck = _starts(nq), _starts(nk)
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), causal=causal, scale=scale)
    rows = torch.tensor([a + i for a, idx in zip(ck, left) for i in idx], device=DEV)
    kl, vl, cl = k[rows], v[rows], _starts([len(i) for i in left])
    G = q.shape[1] // k.shape[1]
    for h in heads:
        o, bound = O.attention(q[:, h:h + 1], kl[:, h // G:h // G + 1], vl[:, h // G:h // G + 1], cq, cl, causal, scale)
        y = got[:, h:h + 1].cpu().double()
        assert bool(torch.isfinite(y).all()), f"{what}: head {h}: {int((~torch.isfinite(y)).sum())} values not finite"
        worst = float(((y - o).abs() / bound.clamp_min(1e-300)).max())
        assert worst <= 1.0, f"{what}: head {h}: error {worst:.2f} of its bound"
    return got


def _low(kind, dtype):
    return -math.inf if kind == "inf" else torch.finfo(dtype).min


RANGES = [(0, 32), (0, 33), (0, 64), (0, 200), (32, 64), (64, 128), (96, 160), (128, 300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["inf", "lowest"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64), (4, 1, 80)])
def test_masked_keys_of_a_few_rows(gpu_lib, pkg, H, Hk, d, causal, kind, dtype):
    # single and few new rows on caches, the masked keys first or in the first block of a later wave
    nq, nk = [1, 1, 3, 5, 2], [40, 65, 300, 301, 700]
    for a, b in RANGES:
        bad = [i for i in range(a, b)]
        for scale in (d ** -0.5, 1.0):
            q, k, v, left = _masked(nq, nk, bad, H, Hk, d, dtype, _low(kind, dtype), seed=a + b)
            # (the last keys of a sequence stay, so that the causal limits do)
            left = [[i for i in range(n) if i in set(idx) or i >= n - 8] for n, idx in zip(nk, left)]
            at = 0
            for n in nk:
                k[at + n - 8:at + n, :, -1] = 0
                at += n
            _check_without(pkg, q, k, v, nq, nk, left, causal, scale, (0, H - 1), f"keys {a} to {b}, scale {scale}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["inf", "lowest"])
def test_masked_keys_of_whole_chunks(gpu_lib, pkg, kind, dtype):
    # one row's keys divided between workgroups, some of which have masked keys alone
    nq, nk, H, Hk, d = [1, 1], [6000, 4100], 8, 2, 128
    assert gpu_lib.packed_attention_workspace_bytes(2, 2, sum(nk), H, Hk, d) > 0
    for a, b in ((0, 2048), (512, 3000), (0, 4090)):
        q, k, v, left = _masked(nq, nk, range(a, b), H, Hk, d, dtype, _low(kind, dtype), seed=a)
        for scale in (d ** -0.5, 1.0):
            _check_without(pkg, q, k, v, nq, nk, left, True, scale, (0, H - 1), f"keys {a} to {b}, scale {scale}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["inf", "lowest"])
@pytest.mark.parametrize("H,Hk,d,nq", [(40, 40, 64, [300, 420, 65]), (32, 8, 128, [500, 300])])
def test_masked_keys_of_many_rows(gpu_lib, pkg, H, Hk, d, nq, kind, dtype):
    for a, b in ((0, 32), (0, 64), (0, 130), (64, 128)):
        # (both ways any keys may be masked, causal the first of a cache that the new rows go on from)
        q, k, v, left = _masked(nq, nq, range(a, min(b, min(nq) - 1)), H, Hk, d, dtype, _low(kind, dtype), seed=b)
        _check_without(pkg, q, k, v, nq, nq, left, False, 1.0, (0, H - 1), f"keys {a} to {b}")
        nk = [n + 200 for n in nq]
        q, k, v, left = _masked(nq, nk, range(a, b), H, Hk, d, dtype, _low(kind, dtype), seed=b)
        _check_without(pkg, q, k, v, nq, nk, left, True, 1.0, (0, H - 1), f"cached keys {a} to {b}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,d,nq,nk", [(8, 2, 128, [1, 3], [70, 300]), (8, 2, 128, [1, 1], [6000, 9]),
                                          (40, 40, 64, [300, 420], [300, 420]), (8, 2, 128, [90], [90])])
def test_rows_that_see_masked_keys_alone(gpu_lib, pkg, H, Hk, d, nq, nk, causal, dtype):
    # scores of -inf: nothing is left, 0 as where no key is seen; the type's lowest value: all are equal, their mean
    q, k, v, _ = _masked(nq, nk, range(max(nk)), H, Hk, d, dtype, -math.inf)
    for scale in (d ** -0.5, 1.0):
        got = pkg.kernels.packed_attention(q, k, v, _cu(_starts(nq)), _cu(_starts(nk)), causal=causal, scale=scale)
        assert bool((got == 0).all())
    if dtype is torch.bfloat16:  # (fp16's lowest leaves the other values' part of the score its own)
        k[..., -1] = torch.finfo(dtype).min
        got = pkg.kernels.packed_attention(q, k, v, _cu(_starts(nq)), _cu(_starts(nk)), causal=causal, scale=1.0)
        zero = torch.zeros_like(q)
        for h in (0, H - 1):
            g = h // (H // Hk)
            o, bound = O.attention(zero[:, :1], k[:, g:g + 1] * 0, v[:, g:g + 1], _starts(nq), _starts(nk), causal, 1.0)
            y = got[:, h:h + 1].cpu().double()
            assert bool(torch.isfinite(y).all()) and float(((y - o).abs() / bound).max()) <= 1.0


def test_leading_masked_keys_of_a_causal_prompt(gpu_lib, pkg):
    # left padding within the prompt itself: the padded rows see nothing (0), the others their own part
    for H, Hk, d, n, pad in ((8, 2, 128, 200, 70), (40, 40, 64, 700, 333), (4, 4, 64, 33, 32)):
        q, k, v, left = _masked([n], [n], range(pad), H, Hk, d, torch.bfloat16, -math.inf, seed=n)
        got = _check_without(pkg, q, k, v, [n], [n], left, True, d ** -0.5, (0, H - 1))
        assert bool((got[:pad] == 0).all())


def test_infinite_and_missing_scores_stay_what_the_formula_makes_them(gpu_lib, pkg):
    # +inf and NaN among the seen scores make the row NaN, beside masked keys too
    for nq, nk, H, Hk in ((1, 300, 8, 2), (600, 600, 40, 40)):
        for bad, kind in ((math.inf, "+inf"), (math.nan, "nan")):
            q, k, v, _ = _masked([nq], [nk], range(64), H, Hk, 64, torch.bfloat16, -math.inf)
            k[150, 0, -1] = bad
            got = pkg.kernels.packed_attention(q, k, v, _cu([0, nq]), _cu([0, nk]))
            G = H // Hk
            assert bool(got[:, :G].isnan().all()) and bool(torch.isfinite(got[:, G:]).all()), kind


# ---- scores of any size ----------------------------------------------------------------------------------

FORMS = [(2, 300, 8, 2, 128), (1, 5000, 8, 2, 128), (600, 600, 40, 40, 64), (5, 40, 4, 1, 80)]  # rows, keys, heads, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2", [8, 10, 11, 16, 20, 22])
@pytest.mark.parametrize("nq,nk,H,Hk,d", FORMS)
def test_a_common_part_of_all_scores_changes_nothing(gpu_lib, pkg, nq, nk, H, Hk, d, log2, sign, dtype):
    # scores 2^log2 + 0 .. 5, all exact in fp32: the softmax is that of 0 .. 5. Where m c stays below its limit of 1,024,
    # its rounding and the FMA's are 2^-24 of that each, on p and on the sum of p: 4 ln 2 2^-14 < 2^-12 of o (values in 1 .. 2)
    g = torch.Generator().manual_seed(log2)
    half = log2 // 2
    q, k = torch.zeros(nq, H, d, dtype=dtype), torch.zeros(nk, Hk, d, dtype=dtype)
    q[..., 0], q[..., 1] = sign * 2.0 ** half, 1
    k[..., 0], k[..., 1] = 2.0 ** (log2 - half), torch.randint(0, 6, (nk, Hk), generator=g).to(dtype)
    v = (1 + torch.rand(nk, Hk, d, generator=g)).to(dtype)
    q, k, v = (t.to(DEV) for t in (q, k, v))
    got = pkg.kernels.packed_attention(q, k, v, _cu([0, nq]), _cu([0, nk]), scale=1.0)
    near = k.clone()
    near[..., 0] = 0
    for h in (0, H - 1):
        e = h // (H // Hk)
        o, bound = O.attention(q[:1, h:h + 1], near[:, e:e + 1], v[:, e:e + 1], [0, 1], [0, nk], False, 1.0)
        err = (got[:, h:h + 1].cpu().double() - o).abs()
        assert float((err / (bound + 2.0 ** -12 * o.abs())).max()) <= 1.0


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2", [12, 30, 40, 64, 100, 120])
@pytest.mark.parametrize("nq,nk,H,Hk,d", FORMS)
def test_far_scores_leave_the_largest_alone(gpu_lib, pkg, nq, nk, H, Hk, d, log2, sign):
    # scores of +-(64 .. 69) 2^log2, exact in fp32, at least 2^12 apart: the mean of the keys of the largest
    g = torch.Generator().manual_seed(log2)
    q, k = torch.zeros(nq, H, d).bfloat16(), torch.zeros(nk, Hk, d).bfloat16()
    q[..., 0] = sign * 2.0 ** (log2 // 2)
    of = torch.randint(64, 70, (nk,), generator=g)
    k[..., 0] = (of * 2.0 ** (log2 - log2 // 2)).bfloat16()[:, None]
    v = torch.randn(nk, Hk, d, generator=g).bfloat16()
    q, k, v = (t.to(DEV) for t in (q, k, v))
    for scale in (1.0, 0.125):
        got = pkg.kernels.packed_attention(q, k, v, _cu([0, nq]), _cu([0, nk]), scale=scale)
        top = (of == (of.max() if sign > 0 else of.min())).nonzero()[:, 0].to(DEV)
        for h in (0, H - 1):
            e = h // (H // Hk)
            o, bound = O.attention(q[:1, h:h + 1] * 0, k[top, e:e + 1] * 0, v[top, e:e + 1], [0, 1], [0, len(top)], False, 1.0)
            err = (got[:, h:h + 1].cpu().double() - o).abs()
            assert float((err / bound).max()) <= 1.0


# ---- probabilities far below their row's largest ---------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nats", [8, 12, 14, 15, 16, 17, 18])
@pytest.mark.parametrize("nq,nk,H,Hk,d,first", [(1, 16384, 4, 1, 128, 0), (1, 16384, 4, 4, 64, 9000), (1, 3000, 4, 4, 64, 0),
                                                (600, 4000, 40, 40, 64, 0), (130, 4000, 32, 8, 128, 3000)])
def test_many_small_probabilities_beside_a_large_one(gpu_lib, pkg, nq, nk, H, Hk, d, first, nats, dtype):
    # one key far above thousands of equal others: with its values 0 the others' are the whole output, and with all
    # values 1 the output is 1, as the sum of the probabilities is that of the products
    g = torch.Generator().manual_seed(nats)
    q, k = torch.zeros(nq, H, d, dtype=dtype), torch.zeros(nk, Hk, d, dtype=dtype)
    q[..., 0], k[first, :, 0] = 1, nats
    v = (1 + 0.5 * torch.randn(nk, Hk, d, generator=g)).to(dtype)
    v[first] = 0
    q, k, v = (t.to(DEV) for t in (q, k, v))
    cq, ck = [0, nq], [0, nk]
    got = pkg.kernels.packed_attention(q, k, v, _cu(cq), _cu(ck), scale=1.0)
    o, bound = O.attention(q[:1, :1], k[:, :1], v[:, :1], [0, 1], ck, False, 1.0)
    y = got[:, :1].cpu().double()
    worst = float(((y - o).abs() / bound).max())
    assert worst <= 1.0, f"{nats} nats: error {worst:.2f} of its bound, {float((y - o).abs().max() / o.abs().max()):.4f} of the largest"
    ones = pkg.kernels.packed_attention(q, k, torch.ones_like(v), _cu(cq), _cu(ck), scale=1.0).double()
    # numerator and sum are the same sums of the same numbers, each within nk + 64 roundings of 2^-24
    assert float((ones - 1).abs().max()) <= O.HALF_STEP[dtype] + 2 * (nk + 64) * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", [0.02, 0.08, 0.3])
@pytest.mark.parametrize("nq,H,Hk,d", [(2, 4, 1, 128), (600, 40, 40, 64)])
def test_scores_that_rise_all_the_way(gpu_lib, pkg, nq, H, Hk, d, step, dtype):
    # the row's maximum moves in every block by less and by more than what it is rescaled for; large values
    nk = 700
    q, k = torch.zeros(nq, H, d, dtype=dtype), torch.zeros(nk, Hk, d, dtype=dtype)
    q[..., :2], k[..., 0] = 1, (step * torch.arange(nk)).to(dtype)[:, None]
    v = (1000 * torch.randn(nk, Hk, d, generator=torch.Generator().manual_seed(1))).to(dtype)
    q, k, v = (t.to(DEV) for t in (q, k, v))
    for causal in (False, True):
        got = pkg.kernels.packed_attention(q, k, v, _cu([0, nq]), _cu([0, nk]), causal=causal, scale=1.0)
        rows = sorted({0, nq // 2, nq - 1})
        for h in (0, H - 1):
            for i in rows:  # (row by row: a row sees the keys up to its own)
                n = i + nk - nq + 1 if causal else nk
                g = h // (H // Hk)
                o, bound = O.attention(q[i:i + 1, h:h + 1], k[:n, g:g + 1], v[:n, g:g + 1], [0, 1], [0, n], False, 1.0)
                y = got[i:i + 1, h:h + 1].cpu().double()
                assert float(((y - o).abs() / bound).max()) <= 1.0


@pytest.mark.parametrize("scale", [1e-37, 1e-42])
@pytest.mark.parametrize("nq,nk,H,Hk,d", FORMS)
def test_scales_of_next_to_nothing_leave_the_mean(gpu_lib, pkg, nq, nk, H, Hk, d, scale):
    # all exponents are 0 to fp32, below its normal range too: the oracle on queries of 0
    g = torch.Generator().manual_seed(nk)
    q, k, v = (torch.randn(n, h, d, generator=g).half().to(DEV) for n, h in ((nq, H), (nk, Hk), (nk, Hk)))
    got = pkg.kernels.packed_attention(q, k, v, _cu([0, nq]), _cu([0, nk]), scale=scale)
    o, bound = O.attention(q[:1, :1] * 0, k[:, :1], v[:, :1], [0, 1], [0, nk], False, 1.0)
    assert float(((got[:, :1].cpu().double() - o).abs() / bound).max()) <= 1.0


# ---- the same call again, and over its queries -----------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,nk,H,Hk,d", [([1, 1], [6000, 4100], 8, 2, 128), ([2, 1, 1], [900, 1, 5000], 4, 4, 64),
                                          ([300, 420, 65], [300, 420, 65], 40, 40, 64), ([24], [24], 40, 40, 64)])
def test_repeats_and_outputs_over_the_queries(gpu_lib, pkg, nq, nk, H, Hk, d, dtype):
    # sums in one order whatever runs beside them; keys divided between workgroups, whose join writes over the queries
    g = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(sum(n), h, d, generator=g).to(dtype).to(DEV) for n, h in ((nq, H), (nk, Hk), (nk, Hk)))
    cq, ck = _cu(_starts(nq)), _cu(_starts(nk))
    ref = pkg.kernels.packed_attention(q, k, v, cq, ck, causal=True)
    for _ in range(4):
        assert torch.equal(pkg.kernels.packed_attention(q, k, v, cq, ck, causal=True), ref)
    over = q.clone()
    assert pkg.kernels.packed_attention(over, k, v, cq, ck, causal=True, out=over) is over and torch.equal(over, ref)
