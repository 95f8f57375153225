"""Build libkvc.so (all HIP sources of csrc/) for gfx950 with hipcc, and the Python
binding of some of its entries (csrc/bind.cpp) with g++ against torch's headers.  The library
needs neither torch nor g++; without the binding the ops that use it take a longer way.

Compiled in-tree so that they travel with the repository:
    gpu_offloading_amd/lib/libkvc.so
    gpu_offloading_amd/lib/kvc_bind.so
Flags: -O3, C++17, gfx950 only, packed-FP32 instruction selection disabled
(``-Xclang -target-feature -Xclang -packed-fp32-ops``; hipcc's host pass
warns that it does not know the feature, which is harmless).
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libkvc.so")
ARCH = "gfx950"

HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


def hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required to build libkvc.so)")


STAMP_PATH = LIB_PATH + ".srchash"

BIND_SRC = os.path.join(CSRC, "bind.cpp")
BIND_PATH = os.path.join(LIB_DIR, "kvc_bind.so")
BIND_STAMP_PATH = BIND_PATH + ".srchash"
BIND_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-Wall"]


def _bind_command(out: str) -> list[str]:
    """g++ line of the binding: Python's and torch's headers, torch's libraries (loaded
    already wherever the binding is)."""
    import importlib.util
    import sysconfig

    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise RuntimeError("torch is not installed")
    torch_dir = os.path.dirname(spec.origin)
    includes = [sysconfig.get_paths()["include"], INCLUDE, os.path.join(torch_dir, "include"),
                os.path.join(torch_dir, "include", "torch", "csrc", "api", "include")]
    return ["g++", *BIND_FLAGS, *(f"-I{p}" for p in includes), BIND_SRC, "-o", out,
            "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _hash(files: list[str], *words: str) -> str:
    import hashlib

    h = hashlib.sha256()
    for path in files:
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(words).encode())
    return h.hexdigest()


def source_hash() -> str:
    """SHA-256 of everything libkvc.so is built from (sources, headers,
    flags): a library whose stamp differs was built from other sources."""
    return _hash(sources() + sorted(glob.glob(os.path.join(CSRC, "*.h"))) +
                 [os.path.join(INCLUDE, "kvc.h")], *HIP_FLAGS)


def binding_hash() -> str:
    """The binding's own: its source, the C ABI that it calls, and the torch and the Python whose
    C++ and C interfaces it was built against."""
    import torch

    return _hash([BIND_SRC, os.path.join(INCLUDE, "kvc.h")], *BIND_FLAGS, torch.__version__,
                 str(torch.version.git_version), sys.version)


def _run(cmd: list[str]) -> tuple[int, list[str]]:
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "'-packed-fp32-ops' is not a recognized feature"
    return res.returncode, [ln for ln in (res.stdout + res.stderr).splitlines()
                            if noise not in ln]


def _build_binding(verbose: bool) -> str | None:
    """Compile the binding (always recompiles); returns why that failed, or None."""
    tmp = BIND_PATH + ".tmp"
    for path in (BIND_PATH, BIND_STAMP_PATH):
        if os.path.exists(path):
            os.remove(path)
    try:
        cmd = _bind_command(tmp)
        if verbose:
            print(" ".join(cmd), flush=True)
        rc, msgs = _run(cmd)
        if rc != 0:
            return "\n".join(msgs)
        if verbose and msgs:
            print("\n".join(msgs), file=sys.stderr)
        stamp = binding_hash()
    except (OSError, RuntimeError, ImportError) as e:      # no g++, no torch
        return str(e)
    os.replace(tmp, BIND_PATH)
    with open(BIND_STAMP_PATH, "w") as f:
        f.write(stamp + "\n")
    return None


def build_library(verbose: bool = False, jobs: int | None = None) -> str:
    """Compile every csrc/*.hip into libkvc.so (always recompiles): one hipcc
    process per source file, in parallel, then one link.  The binding is compiled behind them;
    where it cannot be (no torch, no g++), the library is built all the same and stderr
    says why."""
    from concurrent.futures import ThreadPoolExecutor

    os.makedirs(LIB_DIR, exist_ok=True)
    obj_dir = os.path.join(LIB_DIR, "obj")
    os.makedirs(obj_dir, exist_ok=True)
    srcs = sources()
    objs = [os.path.join(obj_dir, os.path.basename(s)[:-4] + ".o") for s in srcs]
    cmds = [[hipcc(), *HIP_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", s, "-o", o]
            for s, o in zip(srcs, objs)]
    jobs = jobs or min(len(cmds), max(1, min(os.cpu_count() or 1, 16)))
    if verbose:
        for c in cmds:
            print(" ".join(c), flush=True)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        results = list(ex.map(_run, cmds))
    failed = [(s, m) for s, (rc, m) in zip(srcs, results) if rc != 0]
    if failed:
        raise RuntimeError("hipcc failed:\n" + "\n".join(
            f"{s}:\n" + "\n".join(m) for s, m in failed))
    msgs = [ln for _, m in results for ln in m]
    tmp = LIB_PATH + ".tmp"
    link = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    if verbose:
        print(" ".join(link), flush=True)
    rc, lm = _run(link)
    if rc != 0:
        raise RuntimeError("hipcc link failed:\n" + "\n".join(lm))
    msgs += lm
    if verbose and msgs:
        print("\n".join(msgs), file=sys.stderr)
    os.replace(tmp, LIB_PATH)
    with open(STAMP_PATH, "w") as f:
        f.write(source_hash() + "\n")
    why = _build_binding(verbose)
    if why is not None:
        print(f"{BIND_SRC} is not built, the quantised ops do without it: {why}", file=sys.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(verbose=True))
