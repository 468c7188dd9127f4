"""Build the B200 KV block store library (libkvs_b200.so) in-tree for sm_100a.

    python tt-infinity_b200/build.py [--debug]

Compiles csrc/*.cu and csrc/*.cpp with nvcc into kvcache_manager/libkvs_b200.so (the C ABI of
include/kvs.h). nvcc cross-compiles for sm_100a without a GPU.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "kvcache_manager" / "libkvs_b200.so"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cpp"))


def needs_build(out: Path) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    deps = sources() + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.hpp")) + [ROOT / "include" / "kvs.h"]
    return any(p.stat().st_mtime > t for p in deps)


FAST_SRC = CSRC / "pyext" / "kvs_fastcall.c"


def fastcall_path() -> Path:
    import sysconfig

    return PKG / "kvcache_manager" / ("_fastcall" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_fastcall(force: bool = False) -> Path:
    """The CPython module of the block calls' hot path (gcc; it calls the library through
    function pointers, so it does not link against it)."""
    import sysconfig

    import numpy as np

    out = fastcall_path()
    if not force and out.exists() and out.stat().st_mtime > FAST_SRC.stat().st_mtime:
        return out
    cc = os.environ.get("CC", "gcc")
    cmd = [cc, "-O2", "-shared", "-fPIC", "-Wall", "-I", sysconfig.get_paths()["include"], "-I", np.get_include(),
           str(FAST_SRC), "-o", str(out) + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("gcc failed building the _fastcall module")
    os.replace(str(out) + ".tmp", out)
    return out


OPCALL_SRC = CSRC / "pyext" / "kvs_opcall.cpp"


def opcall_path() -> Path:
    import sysconfig

    return PKG / "kvcache_manager" / ("_opcall" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_opcall(force: bool = False) -> Path:
    """The CPython module of the operators on a paged cache (g++ against torch's headers and
    libraries, which the package's import of torch has loaded; it calls libkvs_b200.so through
    function pointers)."""
    import sysconfig

    out = opcall_path()
    try:
        import torch
    except ImportError:  # the operators take torch tensors: nothing to build for
        return out
    if torch.version.cuda is None or not (Path(torch.__file__).parent / "lib" / "libc10_cuda.so").exists():
        return out  # nor without torch's CUDA part
    deps = [OPCALL_SRC, ROOT / "include" / "kvs.h", Path(torch.__file__)]
    if not force and out.exists() and all(d.stat().st_mtime < out.stat().st_mtime for d in deps):
        return out
    home = Path(torch.__file__).parent
    cuda = Path(NVCC).resolve().parents[1]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", sysconfig.get_paths()["include"], "-I", str(ROOT / "include"), "-isystem", str(home / "include"),
           "-isystem", str(home / "include" / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda / "include"),
           str(OPCALL_SRC), "-o", str(out) + ".tmp", "-L", str(home / "lib"), "-ltorch_python", "-ltorch_cpu",
           "-lc10_cuda", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building the _opcall module")
    os.replace(str(out) + ".tmp", out)
    return out


def build(debug: bool = False, verbose: bool = False, force: bool = False) -> Path:
    """The library first: it needs neither Python's nor torch's headers."""
    if force or needs_build(OUT):
        build_library(debug, verbose)
    build_fastcall(force)
    build_opcall(force)
    return OUT


def build_library(debug: bool = False, verbose: bool = False) -> None:
    flags = ARCH + [
        "-std=c++17",
        "--threads", "0",  # compile the sources side by side
        "-lineinfo",
        "-O0" if debug else "-O3",
        "-Xcompiler", "-fPIC,-Wall,-Wno-unused-function",
        "-shared",
        "-I", str(ROOT / "include"),
        "-I", str(CSRC),
        "-o", str(OUT) + ".tmp",
    ]
    if verbose:
        flags += ["-Xptxas", "-v"]
    cmd = [NVCC, *flags, *map(str, sources())]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libkvs_b200.so")
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(str(OUT) + ".tmp", OUT)


if __name__ == "__main__":
    build(debug="--debug" in sys.argv, verbose="-v" in sys.argv, force=True)
    print(OUT)
