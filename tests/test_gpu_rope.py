"""Norm and rotation of queries and keys against a 64-bit restatement, with bounds from the arithmetic."""

import pytest
import torch

from oracle import packed as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]


def _inputs(T, H, Hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = (3 * torch.randn(T, (H + 2 * Hk) * d, generator=g) + 0.5).to(dtype).to(DEV)
    q, k, _ = qkv.split([H * d, Hk * d, Hk * d], dim=1)
    return q.unflatten(1, (H, d)), k.unflatten(1, (Hk, d))


def _weights(H, Hk, d, each, seed=1):
    g = torch.Generator().manual_seed(seed)
    return tuple((1 + 0.3 * torch.randn((h * d) if each else d, generator=g)).to(DEV) for h in (H, Hk))


def _check(got, ref):
    o, bound = ref
    worst = float(((got.detach().cpu().double() - o).abs() / bound).max())
    assert worst <= 1.0, f"error {worst:.2f} of its bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm,over,each", [(None, "head", False), ("rms", "head", False), ("layer", "head", True),
                                            ("rms", "row", True), ("layer", "row", True), ("layer", "row", False)])
@pytest.mark.parametrize("H,Hk,d,rot,interleaved", [(4, 2, 64, 64, False), (32, 8, 128, 64, True), (3, 1, 80, 80, False),
                                                    (5, 5, 72, 48, True), (2, 1, 256, 128, False), (1, 1, 8, 0, False),
                                                    (40, 40, 64, 64, False), (9, 3, 24, 16, True)])
def test_against_the_definition(gpu_lib, pkg, H, Hk, d, rot, interleaved, norm, over, each, dtype):
    T = 7
    q, k = _inputs(T, H, Hk, d, dtype, seed=H + d)
    wq, wk = _weights(H, Hk, d, each)
    rotary = pkg.rotary.Rotary(d, base=10000.0, rot_dim=rot, interleaved=interleaved)
    pos = torch.tensor([0, 1, 17, 4096, 999999, 2 ** 31 - 1, 12345], dtype=torch.int32)
    got = rotary(q, k, pos.to(DEV), norm=norm, over=over, q_w=wq, k_w=wk, eps=1e-5)
    for y, x, w in zip(got, (q, k), (wq, wk)):
        _check(y, O.norm_rope(x, w, pos, rotary.freq, rotary.gain, rot, interleaved, norm, over, 1e-5))


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 8.0}, {"kind": "ntk", "factor": 4.0},
                                     {"kind": "bands", "factor": 8.0, "context": 8192},
                                     {"kind": "yarn", "factor": 16.0, "context": 4096}])
def test_stretched_contexts(gpu_lib, pkg, scaling):
    q, k = _inputs(33, 8, 2, 128, torch.float16)
    rotary = pkg.rotary.Rotary(128, base=500000.0, scaling=scaling)
    pos = torch.arange(33, dtype=torch.int64) * 40009
    got = rotary(q, k, pos.to(DEV), norm="rms")
    for y, x in zip(got, (q, k)):
        _check(y, O.norm_rope(x, None, pos, rotary.freq, rotary.gain, 128, False, "rms", "head", 1e-6))


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_positions_before_zero_and_past_32_bits(gpu_lib, pkg, wide):
    q, k = _inputs(5, 8, 2, 64, torch.bfloat16, seed=9)
    rotary = pkg.rotary.Rotary(64)
    far = 2 ** 31 - 1 if wide is torch.int32 else 2 ** 34 + 5
    pos = torch.tensor([-1, -77, -far, 0, far], dtype=wide)
    got = rotary(q, k, pos.to(DEV))
    for y, x in zip(got, (q, k)):
        _check(y, O.norm_rope(x, None, pos, rotary.freq, rotary.gain, 64, False, None, "head", 1e-6))


@pytest.mark.parametrize("T", [1, 2, 513, 2000])
def test_row_counts_default_positions_and_in_place(gpu_lib, pkg, T):
    q, k = _inputs(T, 32, 4, 64, torch.bfloat16, seed=T)
    rotary = pkg.rotary.Rotary(64)
    got = rotary(q, k, norm="rms")
    pos = torch.arange(T)
    for y, x in zip(got, (q, k)):
        _check(y, O.norm_rope(x, None, pos, rotary.freq, 1.0, 64, False, "rms", "head", 1e-6))
    same = rotary(q, k, pos.to(DEV), norm="rms", out=(q, k))
    assert same[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])


@pytest.mark.parametrize("H,Hk,d,rot,interleaved", [(40, 40, 64, 64, False), (40, 40, 64, 32, True), (7, 3, 128, 128, False),
                                                    (20, 4, 80, 80, False), (90, 10, 64, 64, False), (1, 1, 128, 128, False)])
@pytest.mark.parametrize("norm,over", [("rms", "row"), ("layer", "row"), ("layer", "head"), ("rms", "head"), (None, "head")])
def test_many_rows_in_place_far_from_zero(gpu_lib, pkg, H, Hk, d, rot, interleaved, norm, over):
    # several groups of heads a wave, waves with heads of both and of neither, means many times the spread, every head
    # written over its input; with the weights of both, of one and of neither
    T = 515
    wq, wk = _weights(H, Hk, d, True)
    rotary = pkg.rotary.Rotary(d, rot_dim=rot, interleaved=interleaved)
    pos = torch.arange(T, dtype=torch.int32) * 3
    for w in ((wq, wk), (wq, None), (None, None)):
        q, k = _inputs(T, H, Hk, d, torch.float16, seed=d)
        q, k = q.clone() + 60, k.clone() - 40
        refs = [O.norm_rope(x, v, pos, rotary.freq, rotary.gain, rot, interleaved, norm, over, 1e-5)
                for x, v in zip((q, k), w if norm else (None, None))]
        rotary(q, k, pos.to(DEV), norm=norm, over=over, q_w=w[0], k_w=w[1], eps=1e-5, out=(q, k))
        for y, ref in zip((q, k), refs):
            _check(y, ref)


def test_rows_of_zeros_and_of_infinities(gpu_lib, pkg):
    q, k = _inputs(3, 4, 4, 64, torch.float16)
    q[0], q[1, 2, 5], k[2, 1, 0] = 0, float("inf"), float("nan")
    rotary = pkg.rotary.Rotary(64)
    y, z = rotary(q, k, norm="rms", eps=0.0)
    assert bool(y[0].isnan().all())  # 0 / 0, as the formula has it
    y, z = rotary(q, k, norm="rms", eps=1e-6)
    assert bool((y[0] == 0).all()) and bool(torch.isfinite(y[1, [0, 1, 3]]).all())
    assert bool(z[2, 1].isnan().all()) and bool(torch.isfinite(z[2, [0, 2, 3]]).all())
    y, z = rotary(q, k)  # no norm: only the pair turns bad
    assert int((~torch.isfinite(y)).sum()) == 2 and int(z.isnan().sum()) == 2


def test_graph(gpu_lib, pkg):
    q, k = _inputs(50, 40, 40, 64, torch.float16)
    wq, wk = _weights(40, 40, 64, True)
    rotary = pkg.rotary.Rotary(64)
    ref = rotary(q, k, norm="layer", over="row", q_w=wq, k_w=wk)
    out = tuple(torch.empty_like(t) for t in ref)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary(q, k, norm="layer", over="row", q_w=wq, k_w=wk, out=out)
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


def test_language_model_form(gpu_lib, pkg):
    """Norm over the row, half layout, base 10000, positions from 0: esmc_qk_rope's values in token-major order."""
    B, L, H = 1, 76, 40
    q, k = _inputs(L, H, H, 64, torch.float16, seed=3)
    wq, wk = _weights(H, H, 64, True)
    qkv = torch.cat([q.reshape(L, -1), k.reshape(L, -1), k.reshape(L, -1)], 1).contiguous()
    a, b, _ = pkg.kernels.esmc_qk_rope(qkv, wq, wk, 1e-5, B, L, H)
    y, z = pkg.rotary.Rotary(64)(q, k, norm="layer", over="row", q_w=wq, k_w=wk, eps=1e-5)
    for s, t in ((a, y), (b, z)):
        s = s[0].transpose(0, 1).float()
        # two kernels of the same values: each within its rounding and the fp32 angle of the other (76 x 2^-23)
        assert float((s - t.float()).abs().max()) <= 2 * float(s.abs().max()) * (2.0 ** -11 + 76 * 2.0 ** -23 + 2.0 ** -16)


def test_refusals(gpu_lib, pkg):
    K, E = pkg.kernels, pkg.capi.EsmError
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device=DEV)
    f = torch.ones(32, dtype=torch.float64, device=DEV)

    def refused(code, *a, **kw):
        with pytest.raises(E) as e:
            K.qk_norm_rope(*a, **kw)
        assert e.value.code == code, str(e.value)

    refused(-2, q.float(), q, f)
    refused(-2, q, q.bfloat16(), f)
    refused(-2, q, q[:3], f)
    refused(-2, q, q, f.float())
    refused(-2, q, q, torch.ones(33, dtype=torch.float64, device=DEV))       # more pairs than the head has
    refused(-4, q, q, torch.ones(20, dtype=torch.float64, device=DEV))       # rot 40
    refused(-5, q, q, f.cpu())
    refused(-5, q.cpu(), q, f)
    refused(-2, q, q, f, torch.zeros(3, dtype=torch.int32, device=DEV))
    refused(-2, q, q, f, torch.zeros(4, dtype=torch.float32, device=DEV))
    refused(-4, q, q, f, norm="batch")
    refused(-4, q, q, f, norm="rms", over="all")
    refused(-2, q, q, f, norm="rms", eps=-1.0)
    refused(-2, q, q, f, norm="rms", q_w=torch.ones(65, device=DEV))
    refused(-2, q, q, f, norm="rms", k_w=torch.ones(64, device=DEV, dtype=torch.float16))
    refused(-2, q, q, f, out=(q, q[:, :1]))
    refused(-3, q, q, f, out=(q, q[:1].expand(4, 2, 64)))
    p = torch.zeros_like(q)
    refused(-3, q, p, f, out=(p, q))
    refused(-3, q, p, f, out=(p.clone(), q))
    refused(-3, q[..., 4:36], q[..., 4:36], f[:16])
    refused(-3, p[:, :1], q, f, out=(p.view(-1)[:256].view(4, 1, 64), q))    # over q, other strides
    refused(-3, q, p[:, :1], f, out=(q, p.view(-1)[:256].view(4, 1, 64)))
    w = torch.zeros(1, 520, 256, dtype=torch.float16, device=DEV)
    refused(-4, w, w, f, norm="rms", over="row")
    assert K.qk_norm_rope(q[:0], q[:0], f)[0].shape == (0, 2, 64)
