"""The library's build without torch, and the native module beside it: told apart from one made for another torch or
Python, and done without where it cannot be built or loaded."""

import subprocess
import sys

import pytest
import torch

ALONE = """
import importlib.util, sys
sys.modules["torch"] = None  # as where it is not installed
spec = importlib.util.spec_from_file_location("esm_build", sys.argv[1])
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
assert b.up_to_date(), "the library is current whatever the module is"
assert b.build(force=False) == b.LIB_PATH
b.hipcc = lambda: "true"
b.os.replace = lambda *a: None                  # (nothing is compiled or moved here)
assert b.build(force=True) == b.LIB_PATH        # the library's steps, then the module's, which fail
assert not b.try_build_bind()
"""


def test_the_library_builds_without_torch(pkg):
    pkg.capi.lib(require_gpu=False)
    run = subprocess.run([sys.executable, "-c", ALONE, pkg.build.__file__], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    assert "longer way" in run.stderr


def test_a_module_of_another_environment_is_stale(pkg, monkeypatch):
    b = pkg.build
    pkg.capi.lib(require_gpu=False)
    assert b.bind_up_to_date() and b.bind_environment() == b.environment() != b.source_hash()
    here = b.environment()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert b.environment() != here and not b.bind_up_to_date() and b.up_to_date()
    monkeypatch.undo()
    import sysconfig
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-399")
    assert not b.bind_up_to_date() and b.up_to_date()


def test_calls_take_the_longer_way_without_the_module(pkg, monkeypatch, tmp_path, capsys):
    c, b = pkg.capi, pkg.build
    c.lib(require_gpu=False)

    def fails(*a, **kw):
        raise RuntimeError("no headers")
    monkeypatch.setattr(b, "BIND_PATH", str(tmp_path / "_esm_bind.so"))
    monkeypatch.setattr(b, "bind_command", fails)
    assert c._load_bind() is c._LongWay and "no headers" in capsys.readouterr().err
    assert c._LongWay.qk_norm_rope(1, 2) is c._LongWay.packed_attention() is c._LongWay.f8_linear(3) is None
    # a file that is no module: refused by the loader, not the program's end
    (tmp_path / "_esm_bind.so").write_bytes(b"ESMSRC:" + b.source_hash().encode() + b" ESMENV:" + b.environment().encode())
    monkeypatch.setattr(b, "bind_environment", lambda: b.environment())
    monkeypatch.setattr(b, "library_hash", lambda path=None: b.source_hash())
    assert c._load_bind() is c._LongWay and "cannot be loaded" in capsys.readouterr().err


@pytest.mark.gpu
def test_both_ways_give_the_same_bits(gpu_lib, pkg, monkeypatch):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(70, 640, generator=g).half().cuda()
    qkv = torch.randn(70, 3, 4, 64, generator=g).half().cuda()
    cu, ck = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in ([0, 40, 41, 70], [0, 40, 41, 70]))
    cache = torch.randn(5000, 2, 2, 64, generator=g).half().cuda()
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    end = torch.tensor([0, 5000], dtype=torch.int32, device="cuda")
    lin = pkg.f8.F8Linear.from_float(torch.randn(192, 640, generator=g))
    rotary = pkg.rotary.Rotary(64)

    def run():
        q, k, v = qkv.unbind(1)
        return [*rotary(q, k, norm="rms"), pkg.kernels.packed_attention(q, k, v, cu, ck, causal=True),
                pkg.kernels.packed_attention(q[:1], cache[:, 0], cache[:, 1], one, end, causal=True), lin(x), lin(x[:3])]

    want = run()
    assert pkg.capi.bind is not pkg.capi._LongWay
    monkeypatch.setattr(pkg.capi, "bind", pkg.capi._LongWay)
    assert all(torch.equal(a, b) for a, b in zip(want, run()))


def _outcome(f):
    """A call's tensors, or the code it is refused with."""
    from esmfold2_mlx_amd.capi import EsmError
    try:
        y = f()
    except EsmError as e:
        return e.code
    return [t.clone() for t in y] if isinstance(y, tuple) else [y]


@pytest.mark.gpu
def test_both_ways_take_and_refuse_the_same_calls(gpu_lib, pkg, monkeypatch):
    K, dev = pkg.kernels, "cuda"
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q, kv, cu = r(20, 4, 64).half(), r(20, 2, 64).half(), i32(0, 7, 20)
    wide, f = r(20, 8, 72).half(), torch.rand(32, generator=g, dtype=torch.float64).to(dev)
    codes, scales = (lambda m: (m.codes_packed, m.scales))(pkg.f8.F8Linear.from_float(r(128, 256)))
    x = r(40, 256).bfloat16()
    attention = [(q, kv, kv, cu), (q, kv, kv, cu, None, True, 0.3), (q, kv, kv, cu, cu), (q, kv, kv, i32(0, 3, 9), i32(0, 20, 20)),
                 (wide[:, :4, :64], wide[:, 4:6, :64], wide[:, 6:, :64], cu), (q, wide[:, 4:6, 4:68], kv, cu),
                 (q[:1].expand(20, 4, 64), kv, kv, cu), (q, kv[:, :1].expand(20, 2, 64), kv, cu), (q[:, :3], kv, kv, cu),
                 (q[:1], kv, kv, i32(0, 1), i32(0, 20)), (q[:, :, :60], kv[:, :, :60], kv[:, :, :60], cu), (q, kv.bfloat16(), kv, cu),
                 (q, kv[:5], kv[:5], cu), (q, kv, kv, cu.long()), (q, kv, kv, cu[::2]), (q, kv, kv, i32(0), i32(0)), (q, kv, kv, cu, i32(0, 20)),
                 (q, kv, kv, cu, None, False, 0.0), (q, kv, kv, cu, None, False, float("nan")), (q[:0], kv[:0], kv[:0], i32(0, 0)),
                 (q.float(), kv, kv, cu), (q.cpu(), kv, kv, cu), (q, kv, kv, cu.cpu()), (q[0], kv, kv, cu)]
    rope = [((q, kv, f), {}), ((q, kv, f, torch.arange(20, device=dev)), dict(norm="rms", q_w=r(64), k_w=r(64))),
            ((q, kv, f[:16]), dict(interleaved=True, norm="layer", over="row", q_w=r(256), k_w=r(128))),
            ((q, kv, f, i32(*range(19))), {}), ((q, kv, f, torch.arange(20.0, device=dev)), {}), ((q, kv, f.float()), {}),
            ((q, kv, f[:12]), {}), ((wide[:, :4, :64], wide[:, 4:, 8:], f), dict(norm="rms")), ((q, kv[:5], f), {}),
            ((q, kv, f), dict(norm="rms", q_w=r(63))), ((q, kv, f), dict(q_w=r(63))), ((q, kv, f), dict(norm="rms", eps=-1.0)),
            ((q, kv, f), dict(norm="none")), ((q, kv, f), dict(over="all")), ((q, kv, f[::2]), {}), ((q, kv, f[:0]), dict(norm="layer")),
            ((q[..., 4:36], kv[..., 4:36], f[:16]), {}), ((q, kv.bfloat16(), f), {}), ((q, kv, f), dict(norm="rms", q_w=r(64).half()))]
    linear = [(x, codes, scales, 128), (x[:3], codes, scales, 128), (x[::2], codes, scales, 128), (x[:0], codes, scales, 128),
              (x.t().contiguous().t(), codes, scales, 128), (x[:, :250], codes, scales, 128), (x[:, :128], codes, scales, 128),
              (x.float(), codes, scales, 128), (x, codes, scales, 64), (x, codes, scales.half(), 128), (x, codes.cpu(), scales, 128),
              (x[:1].expand(40, 256), codes, scales, 128), (x[0], codes, scales, 128), (x.half(), codes, scales, 128)]

    def run():
        return ([_outcome(lambda a=a: K.packed_attention(*a)) for a in attention]
                + [_outcome(lambda a=a, kw=kw: K.qk_norm_rope(*a, **kw)) for a, kw in rope]
                + [_outcome(lambda a=a: K.f8_linear(*a)) for a in linear])

    short = run()
    monkeypatch.setattr(pkg.capi, "bind", pkg.capi._LongWay)
    long = run()
    assert {type(a) for a in long} == {int, list}
    written = {3: 9, 15: 0}  # (rows of no sequence hold what was there: not compared)
    for i, (a, b) in enumerate(zip(short, long)):
        if isinstance(a, int) or isinstance(b, int):
            assert a == b, i
        else:
            n = written.get(i)
            assert [t.shape for t in a] == [t.shape for t in b] and all(torch.equal(s[:n], t[:n]) for s, t in zip(a, b)), i
