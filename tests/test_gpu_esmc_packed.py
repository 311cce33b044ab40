"""The language model on packed proteins of different lengths, and on e4m3 linears, against the oracle's block applied
to each protein alone (bars as the padded form's: max|err| <= 1e-2 x RMS of the update or of the state)."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import esmc as oe
from oracle import f8 as of8

pytestmark = pytest.mark.gpu
DEV = "cuda"
LINEARS = ("wqkv", "wo", "w1", "w2")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _weights(D, F_, seed):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    qz = lambda n, k: oe.quantize(r(n, k) * k ** -0.5)  # noqa: E731
    return oe.EsmcBlockWeights(1 + 0.1 * r(D), 0.1 * r(D), 1 + 0.1 * r(D), 1 + 0.1 * r(D), 1 + 0.1 * r(D),
                               0.1 * r(D), qz(3 * D, D), qz(D, D), qz(2 * F_, D), qz(D, F_))


def _block(pkg, p, H):
    lin = {n: pkg.q8.Q8Linear(*(torch.from_numpy(getattr(getattr(p, n), a)) for a in "qsb")) for n in LINEARS}
    return pkg.esmc.EsmcBlock(p.ln1_w, p.ln1_b, p.q_ln, p.k_ln, p.ln2_w, p.ln2_b, *(lin[n] for n in LINEARS), H)


def _model(pkg, D, F_, H, n, seed=10):
    ps = [_weights(D, F_, seed + i) for i in range(n)]
    g = _gen(seed)
    embed, norm_w = torch.randn(33, D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    return pkg.esmc.HipEsmc(embed, [_block(pkg, p, H) for p in ps], norm_w, n_heads=H), ps, embed, norm_w


def _check_alone(hs, ids, ps, embed, norm_w, H):
    x, n = embed.double()[ids][None], len(ps)
    for i, p in enumerate(ps):
        assert float((hs[i].double().cpu() - x[0]).abs().max()) <= 1e-2 * float(x.pow(2).mean().sqrt()) + 1e-6
        x = oe.block_forward(p, x, None, n_heads=H, res_scale=math.sqrt(n / 36), weights="f16")
    last = F.layer_norm(x, x.shape[-1:], norm_w.double(), None, 1e-5)[0]
    assert float((hs[n].double().cpu() - last).abs().max()) <= 1e-2 * float(last.pow(2).mean().sqrt())


@pytest.mark.parametrize("D,F_,H,lengths", [(256, 384, 4, [29, 1, 70, 0, 133]), (640, 640, 10, [200, 65])])
def test_each_protein_as_if_alone(gpu_lib, pkg, D, F_, H, lengths):
    model, ps, embed, norm_w = _model(pkg, D, F_, H, 3)
    g = _gen(2)
    seqs = [torch.randint(0, 33, (L,), generator=g) for L in lengths]
    out = model.packed([s.to(DEV) for s in seqs])
    assert out.hidden_states.shape == (4, sum(lengths), D) and out.lengths == lengths
    assert out.cu_seqlens.tolist() == [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    for hs, ids in zip(out.hidden_states.split(lengths, 1), seqs):
        if len(ids):
            _check_alone(hs, ids, ps, embed, norm_w, H)
    # other members of the batch change nothing that a protein's rows hold (the linears' tiles may, by their roundings)
    alone = model.packed([seqs[0].to(DEV)]).hidden_states
    a, b = out.hidden_states[:, :lengths[0]], alone
    assert float((a - b).abs().max()) <= 1e-2 * float(b.pow(2).mean().sqrt())


def test_real_width_and_positions(gpu_lib, pkg):
    D, F_, H, lengths = 2560, 5120, 40, [90, 33]
    p = _weights(D, F_, seed=5)
    blk = _block(pkg, p, H)
    T, rs = sum(lengths), math.sqrt(80 / 36)
    x = 2 * torch.randn(T, D, generator=_gen(9))
    cu = torch.tensor([0, 90, 123], dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lengths]).to(DEV)
    xd = x.to(DEV)
    h = pkg.kernels.esmc_layer_norm(xd, blk.ln1_w, blk.ln1_b, 1e-5)
    x_out, out = torch.empty_like(xd), torch.empty_like(h)
    rotary = pkg.rotary.Rotary(64)
    blk.run_packed(xd, h, cu, pos, rotary, rs, blk.ln1_w, blk.ln1_b, x_out, out)
    for a, b in ((0, 90), (90, 123)):
        ref = oe.block_forward(p, x[a:b].double()[None], None, n_heads=H, res_scale=rs, weights="f16")[0]
        upd = ref - x[a:b].double()
        err = float((x_out[a:b].double().cpu() - ref).abs().max())
        assert err <= 1e-2 * float(upd.pow(2).mean().sqrt()), err
    # all positions further along: the scores, and so the block, see only differences
    moved = torch.empty_like(x_out)
    blk.run_packed(xd, h, cu, pos + 1000, rotary, rs, blk.ln1_w, blk.ln1_b, moved, out)
    assert float((moved - x_out).abs().max()) <= 1e-2 * float((x_out - xd).pow(2).mean().sqrt())


def test_packed_graph_replay(gpu_lib, pkg):
    model, *_ = _model(pkg, 256, 384, 4, 2)
    ids = torch.randint(0, 33, (150,), generator=_gen(3)).to(DEV)
    cu = torch.tensor([0, 100, 149, 150], dtype=torch.int32, device=DEV)
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


def test_packed_arguments(gpu_lib, pkg):
    model, *_ = _model(pkg, 128, 192, 2, 1)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    for bad in ((torch.zeros(1, 4, dtype=torch.int64), cu), (torch.zeros(4, dtype=torch.int64), cu[None])):
        with pytest.raises(ValueError):
            model.packed_hidden_states(*bad)
    with pytest.raises(ValueError):
        model.packed([])
    with pytest.raises(ValueError):
        model.packed([torch.zeros(1, 4, dtype=torch.int64)])
    assert model.packed([torch.zeros(0, dtype=torch.int64)]).hidden_states.shape == (2, 0, 128)


def test_packed_runs_replaced_parts_or_refuses(gpu_lib, pkg):
    model, *_ = _model(pkg, 128, 192, 2, 2)
    ids = [torch.randint(0, 33, (n,), generator=_gen(n)) for n in (30, 7)]
    want = model.packed(ids).hidden_states
    blk, calls = model.layers[1], []
    ffn = blk.ffn
    blk.ffn = lambda h: (calls.append("ffn"), ffn(h))[1]
    hook = blk.wqkv.register_forward_hook(lambda *a: calls.append("wqkv"))
    assert torch.equal(model.packed(ids).hidden_states, want) and calls == ["wqkv", "ffn"]
    hook.remove()
    attention = blk.attention
    blk.attention = lambda *a: attention(*a)
    with pytest.raises(ValueError):
        model.packed(ids)
    del blk.attention

    class Other(torch.nn.Module):  # another module in the block's place, as hidden_states takes it
        def __init__(self):
            super().__init__()
            self.ln1_w, self.ln1_b, self.ffn, self.attention = blk.ln1_w, blk.ln1_b, blk.ffn, blk.attention
            self.wqkv, self.n_heads = blk.wqkv, blk.n_heads
    model.layers[1] = Other()
    with pytest.raises(ValueError):
        model.packed(ids)


def _f8_reference(p, x, H, rs, dense):
    """oe.block_forward with each linear's input brought to e4m3 as the operator does it."""
    D = x.shape[-1]

    def linear(t, name):
        y, _ = of8.linear(t.half().view(-1, t.shape[-1]), *dense[name])
        return y.view(*t.shape[:-1], -1)

    h = F.layer_norm(x, (D,), p.ln1_w.double(), p.ln1_b.double(), 1e-5)
    q, k, v = linear(h, "wqkv").split(D, dim=-1)
    q, k = (F.layer_norm(t, (D,), w.double(), None, 1e-5) for t, w in ((q, p.q_ln), (k, p.k_ln)))
    heads = lambda t: t.reshape(*t.shape[:2], H, 64).transpose(1, 2)  # noqa: E731
    o = oe.attention(oe.rope(heads(q)), oe.rope(heads(k)), heads(v)).transpose(1, 2).reshape(x.shape)
    x = x + linear(o, "wo") / rs
    h = F.layer_norm(x, (D,), p.ln2_w.double(), p.ln2_b.double(), 1e-5)
    a, b = linear(h, "w1").chunk(2, dim=-1)
    return x + linear(F.silu(a) * b, "w2") / rs


@pytest.mark.parametrize("packed", [False, True])
def test_block_on_e4m3_linears(gpu_lib, pkg, packed):
    D, F_, H, L = 256, 640, 4, 70
    p = _weights(D, F_, seed=3)
    lin = {n: pkg.f8.F8Linear.from_float(getattr(p, n).dense().float()) for n in LINEARS}
    blk = pkg.esmc.EsmcBlock(p.ln1_w, p.ln1_b, p.q_ln, p.k_ln, p.ln2_w, p.ln2_b, *(lin[n] for n in LINEARS), H)
    x = 2 * torch.randn(1, L, D, generator=_gen(4))
    rs = 1.5
    if packed:
        xd = x[0].to(DEV)
        h = pkg.kernels.esmc_layer_norm(xd, blk.ln1_w, blk.ln1_b, 1e-5)
        out = torch.empty_like(xd)
        blk.run_packed(xd, h, torch.tensor([0, L], dtype=torch.int32, device=DEV), torch.arange(L, device=DEV),
                       pkg.rotary.Rotary(64), rs, blk.ln1_w, blk.ln1_b, out, torch.empty_like(h))
        out = out[None]
    else:
        out = blk(x.to(DEV), res_scale=rs)
    dense = {n: (m.codes.cpu(), m.scales.cpu()) for n, m in lin.items()}
    ref = _f8_reference(p, x.double(), H, rs, dense)
    upd = (ref - x.double()).pow(2).mean().sqrt()
    # A value that lies on the border of two e4m3 codes falls to either side by the fp16 roundings before it: one
    # step, 2^-3 of the value at most, of some values in 2^7 (fp16 keeps 7 bits more), in sums of 256 or more; the
    # whole stays far below e4m3's own error of 2^-4 / sqrt(3) = 4 % a value
    err = out.double().cpu() - ref
    assert float(err.pow(2).mean().sqrt()) <= 2e-2 * float(upd)
    with pytest.raises(ValueError):
        blk.params()


def test_from_hf_on_e4m3_linears(gpu_lib, pkg, tmp_path):
    D, F_, H = 128, 256, 2
    g = _gen(21)
    hf = {"esmc.embed_tokens.weight": torch.randn(33, D, generator=g), "esmc.norm.weight": torch.ones(D)}
    for name, shape in {"self_attn.q_proj": (D, D), "self_attn.k_proj": (D, D), "self_attn.v_proj": (D, D),
                        "self_attn.o_proj": (D, D), "mlp.gate_proj": (F_, D), "mlp.up_proj": (F_, D),
                        "mlp.down_proj": (D, F_)}.items():
        hf[f"esmc.layers.0.{name}.weight"] = torch.randn(*shape, generator=g) * shape[1] ** -0.5
    for name in ("input_layernorm", "post_attention_layernorm"):
        hf[f"esmc.layers.0.{name}.weight"], hf[f"esmc.layers.0.{name}.bias"] = torch.ones(D), torch.zeros(D)
    for name in ("q_norm", "k_norm"):
        hf[f"esmc.layers.0.self_attn.{name}.weight"] = torch.ones(D)
    model = pkg.esmc.HipEsmc.from_hf(hf, n_heads=H, linear=pkg.f8.F8Linear)
    assert all(isinstance(getattr(model.layers[0], n), pkg.f8.F8Linear) for n in LINEARS)
    plain = pkg.esmc.HipEsmc.from_hf(hf, n_heads=H)
    ids = torch.randint(0, 33, (40,), generator=g).to(DEV)
    a, b = model(input_ids=ids[None]).hidden_states[-1, 0], plain(input_ids=ids[None]).hidden_states[-1, 0]
    c = model.packed([ids]).hidden_states[-1]
    assert torch.isfinite(a).all()
    # four linears of e4m3 against 8-bit affine ones: some per cent a value, in a LayerNormed output of unit spread
    assert float((a - b).pow(2).mean().sqrt()) <= 0.15 and float((a - c).pow(2).mean().sqrt()) <= 0.03
    with pytest.raises(ValueError):
        pkg.esmc.HipEsmc.from_hf(hf, n_heads=H, linear=pkg.f8.F8Linear, cache=tmp_path / "c.safetensors")
    with pytest.raises(ValueError):
        model.save_cache(tmp_path / "d.safetensors")
