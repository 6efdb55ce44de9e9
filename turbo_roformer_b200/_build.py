"""Build libtrcuda.so in-tree with nvcc for sm_100a (B200), and the frame cache's Python binding.

``python -m turbo_roformer_b200._build`` or ``build()``; the library lands next to this file so that it
travels with the source tree. nvcc cross-compiles: no GPU is needed to build.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB_NAME = "libtrcuda.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
SOURCES = ("api.cu", "tc.cu", "dsp.cu", "pack.cu", "ola_noalloc.cu", "cache.cu")
ARCH_FLAGS = ("-gencode", "arch=compute_100a,code=sm_100a")


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put the CUDA toolkit on PATH)")


def _source_hash() -> str:
    h = hashlib.sha256()
    for d in (CSRC, INCLUDE):
        for name in sorted(os.listdir(d)):
            if name.endswith((".cu", ".cuh", ".h")):
                with open(os.path.join(d, name), "rb") as f:
                    h.update(name.encode())
                    h.update(f.read())
    h.update(" ".join(ARCH_FLAGS).encode())
    return h.hexdigest()[:16]


def _compile(cmd: list[str], path: str, digest: str) -> str:
    """Run a compiler whose output is to be ``path``, and note the sources it was made from. The output gets a name of
    its own until it is whole, so that processes and threads that build at once do not write into each other's."""
    tmp = f"{path}.{os.getpid()}.{threading.get_ident()}.tmp"
    try:
        res = subprocess.run([*cmd, "-o", tmp], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, path)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)
    with open(path + ".hash", "w") as f:
        f.write(digest + "\n")
    return path


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the CUDA sources into ``turbo_roformer_b200/libtrcuda.so`` (skipped when up to date)."""
    stamp = LIB_PATH + ".hash"
    digest = _source_hash()
    if not force and os.path.exists(LIB_PATH) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read().strip() == digest:
                return LIB_PATH
    cmd = [
        _nvcc(),
        *ARCH_FLAGS,
        "-lineinfo",
        "-O3",
        "-std=c++17",
        "-Xcompiler",
        "-fPIC",
        "-shared",
        "-I",
        INCLUDE,
        *(os.path.join(CSRC, s) for s in SOURCES),
    ]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    return _compile(cmd, LIB_PATH, digest)


BINDING_SOURCE = os.path.join(CSRC, "cache_binding.cpp")
BINDING_PATH = os.path.join(HERE, "_cache_binding.so")


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile the frame cache's Python binding (host code against torch's headers; skipped when up to date)."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    sources = b""
    for name in (BINDING_SOURCE, os.path.join(INCLUDE, "trcuda.h")):
        with open(name, "rb") as f:
            sources += f.read()
    digest = hashlib.sha256(sources + f"{torch.__version__} {sys.version}".encode()).hexdigest()[:16]
    stamp = BINDING_PATH + ".hash"
    if not force and os.path.exists(BINDING_PATH) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read().strip() == digest:
                return BINDING_PATH
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    lib = os.path.join(root, "lib")
    cmd = [
        os.environ.get("CXX") or shutil.which("g++") or "c++",
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(f"-I{d}" for d in (os.path.join(root, "include"), os.path.join(root, "include/torch/csrc/api/include"), cuda,
                             sysconfig.get_paths()["include"])),
        BINDING_SOURCE,
        f"-L{lib}",
        "-ltorch_python",
        "-ltorch_cpu",
        "-lc10",
        "-lc10_cuda",
        f"-Wl,-rpath,{lib}",
    ]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    return _compile(cmd, BINDING_PATH, digest)


if __name__ == "__main__":
    print(build_binding(force="--force" in sys.argv, verbose=True))
    print(build(force="--force" in sys.argv, verbose=True))
