"""Build libesmfold2_amd.so (gfx950) in-tree with hipcc.

    python -m esmfold2_mlx_amd.build      (or __graft_entry__.build())

The library is compiled for gfx950 only. Every HIP source is compiled with the
packed-fp32 target feature disabled (-Xclang -target-feature -Xclang
-packed-fp32-ops): the kernels are written without packed fp32 arithmetic and
the compiler must not introduce it. Beside it goes _esm_bind.so, a host-only Python
module against torch's headers (csrc/bind.cpp): the short way into the library for
calls whose host steps would cost more than their kernels. The library needs no torch,
and does not need the module: where that cannot be built the calls take the longer way.
"""

from __future__ import annotations

import hashlib
import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libesmfold2_amd.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
BIND_NAME = "_esm_bind"
BIND_PATH = os.path.join(HERE, BIND_NAME + ".so")
BIND_SOURCE = "bind.cpp"
SOURCES = ["project.hip", "contract.hip", "epilogue.hip", "q8.hip", "transition.hip", "esmc.hip",
           "recycle.hip", "wide.hip", "stream.hip", "rope.hip", "packed.hip",
           "f8.hip", "capi.cpp"]
HEADERS = ["common.h", "kernels.h", os.path.join("..", "..", "include", "esmfold2_amd.h")]
ARCH = "gfx950"


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the HIP library cannot be built")


def source_hash() -> str:
    """sha256 over the names and contents of every source and header the library is built from."""
    h = hashlib.sha256()
    for name in SOURCES + [BIND_SOURCE] + HEADERS:
        h.update(name.encode() + b"\0")
        with open(os.path.join(CSRC, name), "rb") as f:
            h.update(f.read())
    return h.hexdigest()


_TAG = re.compile(rb"ESMSRC:([0-9a-f]{64})")
_ENV_TAG = re.compile(rb"ESMENV:([0-9a-f]{64})")


def _tag(path: str, tag) -> str | None:
    try:
        with open(path, "rb") as f:
            m = tag.search(f.read())
    except OSError:
        return None
    return m.group(1).decode() if m else None


def library_hash(path: str = LIB_PATH) -> str | None:
    """The source hash a built library was compiled from (the ESMSRC tag capi.cpp embeds), or None."""
    return _tag(path, _TAG)


def environment() -> str:
    """sha256 over what the module is compiled against beside its sources: torch's release and C++ ABI, Python's ABI."""
    import sysconfig

    import torch
    parts = (torch.__version__, int(torch._C._GLIBCXX_USE_CXX11_ABI), sysconfig.get_config_var("SOABI"))
    return hashlib.sha256(repr(parts).encode()).hexdigest()


def bind_environment(path: str = BIND_PATH) -> str | None:
    """The environment a built module was compiled in (its ESMENV tag), or None."""
    return _tag(path, _ENV_TAG)


FLAGS = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def compile_command(src: str, obj: str, src_hash: str) -> list[str]:
    """hipcc -c of one source (every HIP source with packed fp32 disabled)."""
    return [hipcc(), *FLAGS, f"-DESM_SOURCE_HASH=\"{src_hash}\"", "-c", os.path.join(CSRC, src), "-o", obj]


def link_command(objs: list[str], out: str) -> list[str]:
    return [hipcc(), f"--offload-arch={ARCH}", "-shared", *objs, "-o", out]


def bind_command(obj: str, src_hash: str) -> list[str]:
    """hipcc -c of the Python module (host code only)."""
    import sysconfig

    import torch
    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    return [hipcc(), "-O2", "-std=c++17", "-fPIC", "-Wall", "-DUSE_ROCM", f"-DESM_SOURCE_HASH=\"{src_hash}\"",
            f"-DESM_ENVIRONMENT=\"{environment()}\"", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + inc,
            "-I" + os.path.join(inc, "torch", "csrc", "api", "include"), "-I" + sysconfig.get_paths()["include"], "-c",
            os.path.join(CSRC, BIND_SOURCE), "-o", obj]


def bind_link_command(obj: str, out: str) -> list[str]:
    """The module's link: torch's libraries are found loaded when it is imported."""
    import torch
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    return [cxx, "-shared", obj, "-o", out, "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-ltorch_python",
            "-ltorch_cpu", "-lc10", "-lc10_hip"]


def up_to_date() -> bool:
    """True when the built library exists and was compiled from the current sources (by content)."""
    return library_hash() == source_hash()


def bind_up_to_date() -> bool:
    """True when the built module exists and was compiled from the current sources, in this environment."""
    return library_hash(BIND_PATH) == source_hash() and bind_environment() == environment()


_NOISE = "is not a recognized feature for this target"  # host pass of the fp32 feature flag


def _run(procs) -> str:
    msgs, failed = [], []
    for cmd, p in procs:
        out, _ = p.communicate()
        text = "\n".join(l for l in out.splitlines() if _NOISE not in l)
        if p.returncode != 0:
            failed.append(f"{' '.join(cmd)}\n{text}")
        elif text.strip():
            msgs.append(text)
    if failed:
        raise RuntimeError("hipcc failed:\n" + "\n".join(failed))
    return "\n".join(msgs)


def _start(cmd: list[str], verbose: bool):
    if verbose:
        print("[build]", " ".join(cmd), flush=True)
    return cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _show(msgs, verbose: bool) -> None:
    if verbose and any(m.strip() for m in msgs):
        print("\n".join(m for m in msgs if m.strip()), flush=True)


def build_library(verbose: bool = False, jobs: int | None = None) -> str:
    """Compile the library: one hipcc -c per source, up to ``jobs`` at a time, then one link into the in-tree .so."""
    import tempfile
    h = source_hash()
    jobs = jobs or max(1, min(len(SOURCES), os.cpu_count() or 1, 16))
    with tempfile.TemporaryDirectory(prefix="esm_build_") as tmpdir:
        objs = [os.path.join(tmpdir, src.replace(".", "_") + ".o") for src in SOURCES]
        pending = [compile_command(src, obj, h) for src, obj in zip(SOURCES, objs)]
        msgs = []
        while pending:
            batch, pending = pending[:jobs], pending[jobs:]
            msgs.append(_run([_start(cmd, verbose) for cmd in batch]))
        tmp = LIB_PATH + ".tmp"
        msgs.append(_run([_start(link_command(objs, tmp), verbose)]))
    _show(msgs, verbose)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_bind(verbose: bool = False) -> str:
    """Compile and link the module. Raises where torch, its headers or Python's are missing, or do not fit."""
    import tempfile
    with tempfile.TemporaryDirectory(prefix="esm_build_") as tmpdir:
        obj, tmp = os.path.join(tmpdir, "bind.o"), BIND_PATH + ".tmp"
        msgs = [_run([_start(bind_command(obj, source_hash()), verbose)])]
        msgs.append(_run([_start(bind_link_command(obj, tmp), verbose)]))
    _show(msgs, verbose)
    os.replace(tmp, BIND_PATH)
    return BIND_PATH


def try_build_bind(verbose: bool = False) -> bool:
    """``build_bind``, its failure reported on stderr rather than raised: whether the module is there."""
    try:
        build_bind(verbose)
    except Exception as e:  # noqa: BLE001  (whatever it is, the library stands without the module)
        print(f"[esmfold2_amd] {BIND_NAME} cannot be built, its calls take the longer way: {e}", file=sys.stderr, flush=True)
        return False
    return True


def build(force: bool = True, verbose: bool = False, jobs: int | None = None) -> str:
    """Compile the library (always when ``force``), then the module beside it. Returns the library's path."""
    if force or not up_to_date():
        build_library(verbose, jobs)
        try_build_bind(verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    sys.exit(0)
