"""Build libgko_b200.so (all CUDA kernels + the C ABI) in-tree with nvcc for sm_100a.

Usage: python -m evocompile_b200.build [--force]
The library lands next to this file so that it travels with the source tree, and so does _gko_torch.so, the
compiled tensor-level host code of binding/ (g++ against torch's headers, linked to the library).
"""

from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
REPO = PKG.parent
LIB = PKG / "libgko_b200.so"
BINDING_SRC = PKG / "binding" / "gko_torch.cpp"
BINDING = PKG / "_gko_torch.so"
BUILD_DIR = REPO / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    return str(Path(cuda) / "bin" / "nvcc")


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _digest() -> str:
    h = hashlib.sha256()
    for p in sorted(list(CSRC.glob("*")) + [REPO / "include" / "gko_b200.h"]):
        if p.is_file():
            h.update(p.name.encode())
            h.update(p.read_bytes())
    h.update(" ".join(ARCH + NVCC_FLAGS).encode())
    return h.hexdigest()[:16]


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every translation unit under csrc/ and link libgko_b200.so. Returns its path."""
    stamp = PKG / ".libgko_b200.stamp"
    digest = _digest()
    if LIB.exists() and stamp.exists() and stamp.read_text().strip() == digest and not force:
        build_binding()
        return LIB
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = BUILD_DIR / (src.name + ".o")
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", str(REPO / "include"), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, pr in procs:
        out, _ = pr.communicate()
        text = out.decode(errors="replace")
        if pr.returncode != 0:
            failed.append(f"--- {src.name}\n{text}")
        elif verbose and text.strip():
            print(text)
    if failed:
        raise RuntimeError("nvcc failed:\n" + "\n".join(failed))
    tmp = LIB.with_suffix(".so.tmp")
    link = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart", "-lcuda"]
    # libcuda is resolved at run time from the driver; link against the stub when present.
    stub = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "lib64" / "stubs"
    if stub.is_dir():
        link[-1:-1] = ["-L", str(stub)]
    r = subprocess.run(link, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    os.replace(tmp, LIB)
    stamp.write_text(digest)
    build_binding(force, verbose)
    return LIB


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile binding/gko_torch.cpp into _gko_torch.so, against this interpreter's torch. Returns its path."""
    import torch

    stamp = PKG / "._gko_torch.stamp"
    h = hashlib.sha256(BINDING_SRC.read_bytes() + (REPO / "include" / "gko_b200.h").read_bytes())
    h.update(f"{torch.__version__} {sys.version}".encode())
    digest = h.hexdigest()[:16]
    if BINDING.exists() and stamp.exists() and stamp.read_text().strip() == digest and not force:
        return BINDING
    home = Path(torch.__file__).resolve().parent
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_gko_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(home / "include"), "-I", str(home / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", str(cuda / "include"), "-I", sysconfig.get_paths()["include"], str(BINDING_SRC), "-o", str(tmp),
           "-L", str(home / "lib"), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_python",
           "-L", str(PKG), "-l:" + LIB.name, "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed:\n" + r.stdout + r.stderr)
    os.replace(tmp, BINDING)
    stamp.write_text(digest)
    return BINDING


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose=True)
    print(p)
