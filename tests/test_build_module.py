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
