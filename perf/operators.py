"""Language-model operators for packed batches, as measurable cases.

A batch of proteins (or of prompts) of different lengths goes through a transformer block without
padding: the rows of all sequences stand behind one another, and ``cu`` holds where each begins.
Three operators carry such a block, and each stands here by itself:

* ``packed_attention``: softmax(q k^T scale) v within each sequence, queries in groups that share a
  key head, both ways or causal (the last query sees the last key, so a single new token sees a
  whole cache);
* ``qk_norm_rope``: the norm of queries and keys, over each head or over the whole row, and the
  rotation of each row's position in the same pass;
* ``F8Linear``: a linear with weights in e4m3, one scale per 128 x 128 block, whose input is
  brought to e4m3 with one scale per row and 128 columns.

``listed()`` holds the fixed cases, ``draw(rng)`` makes one more from the same ranges. ``prepare``
builds inputs on the GPU from the seed, ``run`` is one pass (plain torch, or the package where
``own`` is true), ``exact`` the same by the definition in 64 bits.
"""

import importlib.util
import math
import os
import sys

import torch

own = False

# (query heads, key heads, head size): the language model's own, then grouped forms
HEADS = ((40, 40, 64), (32, 8, 128), (16, 2, 128), (20, 4, 80), (24, 8, 64), (8, 1, 128))
# (K, N): the language model's linears, one ragged in both, and two square ones
LINEARS = ((2560, 7680), (2560, 2560), (2560, 10240), (5120, 2560), (1104, 1608), (4096, 4096), (8192, 8192))
EPS = 1e-5
BLOCK = 128            # values (and weight rows) under one scale
TOP = 448.0            # the largest e4m3 value
FLOOR = 2.0 ** -96     # the least maximum a scale is made for


def _package():
    """The package directory of the working folder (its name has a hyphen), imported as a program
    outside the repository imports it."""
    if "esmfold2_mlx_amd" not in sys.modules:
        root = os.path.abspath("esmfold2-mlx_amd")
        spec = importlib.util.spec_from_file_location("esmfold2_mlx_amd", os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["esmfold2_mlx_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["esmfold2_mlx_amd"]


# ---- the cases ------------------------------------------------------------------------------


def listed():
    return [
        # One step of generation for eight requests: one new token each against caches of very
        # different lengths, grouped heads. Bound by the caches' bytes.
        dict(name="attention-token", kind="attention", heads=1, new="1,1,1,1,1,1,1,1",
             old="16384,9001,4096,2500,1024,333,76,0", causal=True, dtype="bf16"),
        # A peptide through the language model: the smallest call, latency alone.
        dict(name="attention-24", kind="attention", heads=0, new="24", old="0", causal=False, dtype="fp16"),
        # A batch of proteins of the language model, both ways, no padding between them.
        dict(name="attention-proteins", kind="attention", heads=0,
             new="238,76,512,300,24,476,1100,129,1,350,64,211", old="0", causal=False, dtype="fp16"),
        # Prompts of different lengths in one causal batch, one of them continued from a cache.
        dict(name="attention-prompts", kind="attention", heads=1, new="2048,777,4096,1,1301,64",
             old="0,0,0,500,1000,4000", causal=True, dtype="bf16"),
        # One long prompt, causal: bound by the matrix cores.
        dict(name="attention-16384", kind="attention", heads=1, new="16384", old="0", causal=True, dtype="bf16"),
        # Queries and keys of eight new tokens far into their contexts: latency.
        dict(name="rope-token", kind="rope", heads=1, rows=8, far=131072, norm="rms", over="head", rot=128,
             interleaved=False, scaling="bands", dtype="bf16"),
        # The language model's own form: one LayerNorm over the row of all heads, half layout.
        dict(name="rope-proteins", kind="rope", heads=0, rows=3481, far=1100, norm="layer", over="row", rot=64,
             interleaved=False, scaling="none", dtype="fp16"),
        # A long prompt: norm of each head, pairs side by side, half of each head rotated, positions
        # stretched beyond the trained context. Bound by the rows' bytes.
        dict(name="rope-16384", kind="rope", heads=1, rows=16384, far=1000000, norm="rms", over="head", rot=64,
             interleaved=True, scaling="yarn", dtype="bf16"),
        # One token through the widest linear of the language model: the weights' bytes.
        dict(name="linear-1", kind="linear", linear=2, rows=1, dtype="bf16"),
        # The reference protein through the linear that closes the feed-forward half.
        dict(name="linear-238", kind="linear", linear=3, rows=238, dtype="fp16"),
        # A packed batch of proteins through the projection to queries, keys and values.
        dict(name="linear-3481", kind="linear", linear=0, rows=3481, dtype="fp16"),
        # A long prompt through a wide square linear: bound by the matrix cores.
        dict(name="linear-8192", kind="linear", linear=6, rows=8192, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(("attention", "rope", "linear"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "attention":
        heads = rng.randrange(len(HEADS))
        causal = rng.random() < 0.6
        n = _spread(rng, 1, 24)
        if rng.random() < 0.35:  # single tokens against caches
            new, old = [1] * n, [_spread(rng, 1, 16384) - 1 for _ in range(n)]
        else:
            new, old = [_spread(rng, 1, 4096) for _ in range(n)], [0] * n
            if causal and rng.random() < 0.5:
                old = [rng.choice((0, _spread(rng, 1, 4096))) for _ in range(n)]
            while sum(a * (a + b) for a, b in zip(new, old)) > 6e7:
                new, old = new[:-1], old[:-1]
        text = lambda v: ",".join(str(i) for i in v)  # noqa: E731
        return dict(kind=kind, heads=heads, new=text(new), old=text(old), causal=causal, dtype=dtype)
    if kind == "rope":
        heads = rng.randrange(len(HEADS))
        d = HEADS[heads][2]
        return dict(kind=kind, heads=heads, rows=_spread(rng, 1, 16384), far=_spread(rng, 1000, 1000000),
                    norm=rng.choice(("rms", "layer", "none")), over=rng.choice(("head", "row")),
                    rot=rng.choice([r for r in (32, 64, 80, 128) if r <= d]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "ntk", "yarn", "bands")), dtype=dtype)
    return dict(kind=kind, linear=rng.randrange(len(LINEARS)), rows=_spread(rng, 1, 8192), dtype=dtype)


def _type(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _lengths(case):
    """(new rows, keys) of each sequence: its keys are what is in its cache and its new rows."""
    new = [int(v) for v in case["new"].split(",")]
    old = [int(v) for v in case["old"].split(",")]
    if len(old) == 1:
        old = old * len(new)
    return new, [a + b for a, b in zip(new, old)]


def _starts(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _seen(nq, nk, causal):
    """Query and key pairs of one sequence that count."""
    if not causal:
        return nq * nk
    first = nk - nq + 1  # keys the first query sees (nk >= nq here)
    return nq * first + nq * (nq - 1) // 2


def work(case):
    if case["kind"] == "attention":
        H, Hk, d = HEADS[case["heads"]]
        nq, nk = _lengths(case)
        pairs = sum(_seen(a, b, case["causal"]) for a, b in zip(nq, nk))
        return {"bytes": 2 * d * (2 * H * sum(nq) + 2 * Hk * sum(nk)), "flops": 4 * H * d * pairs}
    if case["kind"] == "rope":
        H, Hk, d = HEADS[case["heads"]]
        T = case["rows"]
        return {"bytes": 2 * 2 * T * (H + Hk) * d + 4 * T, "flops": 10 * T * (H + Hk) * d}
    K, N = LINEARS[case["linear"]]
    M = case["rows"]
    return {"bytes": 2 * M * K + N * K + 2 * M * N, "flops": 2 * M * K * N}


# ---- inputs ---------------------------------------------------------------------------------


def _scaling(case):
    """What the rotation of this case is stretched by: a trained context of 8,192 taken 16 times as far."""
    kind = case["scaling"]
    if kind == "none":
        return None
    s = {"kind": kind, "factor": 16.0}
    if kind in ("yarn", "bands"):
        s["context"] = 8192
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _type(case)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    state = dict(case=case)
    if case["kind"] == "attention":
        H, Hk, d = HEADS[case["heads"]]
        nq, nk = _lengths(case)
        # queries and keys as a norm with trained weights leaves them: scores of a few units
        if nq == nk:  # one projection's rows, [queries | keys | values]
            qkv = normal(sum(nq), (H + 2 * Hk) * d)
            qkv[:, :H * d] *= 1.5
            q, k, v = qkv.to(t).split([H * d, Hk * d, Hk * d], dim=1)
        else:  # new rows against a cache
            q, k, v = (1.5 * normal(sum(nq), H * d)).to(t), normal(sum(nk), Hk * d).to(t), normal(sum(nk), Hk * d).to(t)
        cq, ck = _starts(nq), _starts(nk)
        state.update(q=q.unflatten(1, (H, d)), k=k.unflatten(1, (Hk, d)), v=v.unflatten(1, (Hk, d)), starts=(cq, ck),
                     cu_q=torch.tensor(cq, dtype=torch.int32, device="cuda"),
                     cu_k=torch.tensor(ck, dtype=torch.int32, device="cuda"))
    elif case["kind"] == "rope":
        H, Hk, d = HEADS[case["heads"]]
        T = case["rows"]
        qkv = (normal(T, (H + 2 * Hk) * d) * (0.5 + torch.rand(T, 1, generator=g, device="cuda"))).to(t)
        q, k, _ = qkv.split([H * d, Hk * d, Hk * d], dim=1)
        wide = case["over"] == "row"
        wq, wk = (1 + 0.2 * normal(h * d if wide else d) for h in (H, Hk))
        # rows of a batch stand anywhere in their contexts
        first = torch.randint(0, max(1, case["far"] - T), (1,), generator=g, device="cuda")
        pos = ((first + torch.arange(T, device="cuda")) % case["far"]).to(torch.int32)
        state.update(q=q.unflatten(1, (H, d)), k=k.unflatten(1, (Hk, d)), wq=wq, wk=wk, pos=pos)
        if own:
            state["rotary"] = _package().rotary.Rotary(d, base=500000.0, rot_dim=case["rot"],
                                                       interleaved=case["interleaved"], scaling=_scaling(case))
        else:
            state["freq"], state["gain"] = _frequencies(case)
    else:
        K, N = LINEARS[case["linear"]]
        M = case["rows"]
        # activations with a few strong channels, as trained models have them
        x = normal(M, K) * (1 + 9 * (torch.rand(K, generator=g, device="cuda") < 0.01))
        w = normal(N, K) / math.sqrt(K)
        codes, scales = _weights(w)
        state.update(x=x.to(t), codes=codes, scales=scales)
        if own:
            state["linear"] = _package().f8.F8Linear(codes, scales)
    return state


def _weights(w):
    """A trained weight [N, K] brought to e4m3: codes and one scale per 128 x 128 block."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    p = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    p[:N, :K] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    s = p.abs().amax((1, 3)).clamp_min(FLOOR) / TOP
    codes = (p / s[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous().to(torch.float8_e4m3fn)
    return codes, s


# ---- one pass -------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "attention":
        if own:
            return _package().kernels.packed_attention(state["q"], state["k"], state["v"], state["cu_q"],
                                                       state["cu_k"], causal=case["causal"])
        return _attention(state["q"], state["k"], state["v"], state["starts"], case["causal"])
    if kind == "rope":
        if own:
            norm = None if case["norm"] == "none" else case["norm"]
            w = (None, None) if norm is None else (state["wq"], state["wk"])
            return state["rotary"](state["q"], state["k"], state["pos"], norm=norm, over=case["over"], q_w=w[0],
                                   k_w=w[1], eps=EPS)
        return tuple(_norm_rope(x, w, state["pos"], state["freq"], state["gain"], case)
                     for x, w in ((state["q"], state["wq"]), (state["k"], state["wk"])))
    if own:
        return state["linear"](state["x"])
    return _linear(state["x"], state["codes"], state["scales"])


def _attention(q, k, v, starts, causal):
    """Softmax attention in 32 bits, a sequence at a time, as many key heads at once as 8 GB of scores hold."""
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    H, Hk, d = q.shape[1], k.shape[1], q.shape[2]
    G = H // Hk
    for (q0, q1), (k0, k1) in zip(*(zip(c[:-1], c[1:]) for c in starts)):
        nq, nk = q1 - q0, k1 - k0
        if nq == 0 or nk == 0:
            continue
        masked = None
        if causal and nq > 1:
            i = torch.arange(nq, device=q.device)
            masked = torch.arange(nk, device=q.device)[None, :] > (i + (nk - nq))[:, None]
        step = max(1, min(Hk, (1 << 31) // (G * nq * nk)))
        for h in range(0, Hk, step):
            n = min(step, Hk - h)
            kh, vh = (t[k0:k1, h:h + n].float().transpose(0, 1).contiguous() for t in (k, v))
            qh = q[q0:q1, h * G:(h + n) * G].float().transpose(0, 1).reshape(n, G * nq, d)
            s = torch.bmm(qh, kh.transpose(1, 2).contiguous()).view(n, G, nq, nk) * d ** -0.5
            if masked is not None:
                s.masked_fill_(masked, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.bmm(p.view(n, G * nq, nk), vh).view(n * G, nq, d) / p.sum(-1).view(n * G, nq, 1)
            out[q0:q1, h * G:(h + n) * G] = o.transpose(0, 1).to(out.dtype)
    return out


def _frequencies(case):
    """(radians per position of each pair, in 64 bits; the factor on sine and cosine)."""
    rot, base = case["rot"], 500000.0
    s = _scaling(case)
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    if s is not None and s["kind"] == "ntk":
        base *= s["factor"] ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if s is None or s["kind"] == "ntk":
        return f, 1.0
    if s["kind"] == "linear":
        return f / s["factor"], 1.0
    turns = s["context"] * f / (2 * math.pi)  # of this pair within the trained context
    if s["kind"] == "bands":  # pairs of few turns are stretched, of many kept, linear between in the turns
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / s["factor"] * (1 - keep) + f * keep, 1.0
    # yarn: linear between in the pair's index, from the pair of 32 turns to the one of 1 turn
    at = lambda n: rot * math.log(s["context"] / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    keep = 1 - ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / s["factor"] * (1 - keep) + f * keep, 0.1 * math.log(s["factor"]) + 1


def _norm_rope(x, w, pos, freq, gain, case):
    T, H, d = x.shape
    y = x.float()
    if case["norm"] != "none":
        rows = y.reshape(T, H * d) if case["over"] == "row" else y
        if case["norm"] == "layer":
            rows = rows - rows.mean(-1, keepdim=True)
        rows = rows * torch.rsqrt((rows * rows).mean(-1, keepdim=True) + EPS) * w
        y = rows.view(T, H, d)
    angle = pos.double()[:, None] * freq  # far positions: in 64 bits
    cos, sin = (torch.cos(angle) * gain).float()[:, None], (torch.sin(angle) * gain).float()[:, None]
    rot = case["rot"]
    out = y.clone()
    if case["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return out.to(x.dtype)


def _linear(x, codes, scales):
    """x in e4m3 by rows of 128, both sides back to 32 bits, one product."""
    M, K = x.shape
    N, kb = codes.shape[0], scales.shape[1]
    p = torch.zeros(M, kb * BLOCK, device=x.device)
    p[:, :K] = x
    p = p.view(M, kb, BLOCK)
    top = p.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    p = (p * (TOP / top)).to(torch.float8_e4m3fn).float() * (top / TOP)
    w = codes.float() * scales.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    return (p.view(M, kb * BLOCK)[:, :K] @ w.t()).to(x.dtype)


# ---- the definition in 64 bits --------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attention":
        return _attention64(state, case)
    if case["kind"] == "rope":
        return tuple(_rope64(state[a], state[b], state["pos"], case) for a, b in (("q", "wq"), ("k", "wk")))
    return _linear64(state)


def _attention64(state, case):
    q, k, v = (state[n] for n in "qkv")
    cq, ck = state["starts"]
    G, d = q.shape[1] // k.shape[1], q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s in range(len(cq) - 1):
        nq, nk = cq[s + 1] - cq[s], ck[s + 1] - ck[s]
        keys = torch.arange(nk, device=q.device)
        for h in range(q.shape[1]):
            kh = k[ck[s]:ck[s + 1], h // G].double()
            vh = v[ck[s]:ck[s + 1], h // G].double()
            for r in range(0, nq, 4096):  # queries by parts
                n = min(4096, nq - r)
                z = (q[cq[s] + r:cq[s] + r + n, h].double() @ kh.t()) / math.sqrt(d)
                if case["causal"]:
                    last = r + torch.arange(n, device=q.device) + nk - nq
                    z = torch.where(keys <= last[:, None], z, torch.full_like(z, -math.inf))
                out[cq[s] + r:cq[s] + r + n, h] = torch.softmax(z, dim=1) @ vh
    return out


def _rope64(x, w, pos, case):
    T, H, d = x.shape
    rot, base = case["rot"], 500000.0
    y, w = x.double(), w.double()
    if case["norm"] != "none":
        dims = (1, 2) if case["over"] == "row" else (2,)
        if case["norm"] == "layer":
            y = y - y.mean(dims, keepdim=True)
        y = y / torch.sqrt((y ** 2).mean(dims, keepdim=True) + EPS)
        y = y * (w.view(H, d) if case["over"] == "row" else w.view(1, d))
    gain, factor, context = 1.0, 16.0, 8192.0
    freq = []
    kind = case["scaling"]
    for i in range(rot // 2):
        f = math.pow(base * (math.pow(factor, rot / (rot - 2)) if kind == "ntk" else 1.0), -2.0 * i / rot)
        if kind == "linear":
            f /= factor
        elif kind == "bands":
            length = 2 * math.pi / f
            if length > context / 1.0:
                f /= factor
            elif length >= context / 4.0:
                keep = (context / length - 1.0) / 3.0
                f = (1 - keep) * f / factor + keep * f
        elif kind == "yarn":
            gain = 1.0 + math.log(factor) / 10.0
            pair = [rot * math.log(context / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0)]
            low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
            stretch = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = f / factor * stretch + f * (1 - stretch)
        freq.append(f)
    z = torch.polar(torch.full((T, rot // 2), gain, dtype=torch.float64, device=x.device),
                    pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device))[:, None]
    out = y.clone()
    first = slice(0, rot, 2) if case["interleaved"] else slice(0, rot // 2)
    second = slice(1, rot, 2) if case["interleaved"] else slice(rot // 2, rot)
    turned = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
    out[..., first], out[..., second] = turned.real, turned.imag
    return out


def _linear64(state):
    x, codes, scales = state["x"], state["codes"], state["scales"]
    M, K = x.shape
    N = codes.shape[0]
    y = torch.zeros(M, N, dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        cols = slice(b * BLOCK, min(K, (b + 1) * BLOCK))
        xb = x[:, cols].double()
        s = xb.abs().amax(1, keepdim=True).clamp_min(FLOOR) / TOP
        # e4m3's values stand for the codes; 32 bits on the way there, as torch converts from them
        xq = (xb / s).float().to(torch.float8_e4m3fn).double() * s
        wb = codes[:, cols].double() * scales[:, b].double().repeat_interleave(BLOCK)[:N, None]
        y += xq @ wb.t()
    return y
