"""Builds libnnb.so (the HIP kernels + C ABI) in-tree with hipcc for gfx950."""
from __future__ import annotations

import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libnnb.so")

# (source, extra flags).  The tree kernels must not contract a*b+c into an FMA: the
# selection score has to round like the scalar CPython expression it replaces.
SOURCES = [
    ("tree_kernels.hip", ["-ffp-contract=off"]),
    ("net_kernels.hip", []),
    ("net_kernels_f16.hip", []),
    ("net_kernels_split.hip", []),
    ("mx4_kernels.hip", []),
    ("ortho_kernels.hip", []),
    ("nnb_api.hip", []),
]
# Packed float32 instructions are kept out of all kernels: some of their forms have been seen to give wrong results.
COMMON = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; libnnb.so cannot be built")
    return exe


def _stale(target: str, deps: list) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_lib(force: bool = False, verbose: bool = False) -> str:
    hipcc = _hipcc()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "nnb.h"))
    objs, running = [], []                                 # compiled side by side: one source takes half of the time
    for src, extra in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(CSRC, src.replace(".hip", ".o"))
        if force or _stale(o, [s] + headers):
            cmd = [hipcc, *COMMON, *extra, "-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append((cmd, o, subprocess.Popen(cmd)))
        objs.append(o)
    failed = [(cmd, o, p.returncode) for cmd, o, p in running if p.wait() != 0]
    for cmd, o, _ in failed:
        if os.path.exists(o):                              # an older one would pass for its result
            os.remove(o)
    if failed:
        raise subprocess.CalledProcessError(failed[0][2], failed[0][0])
    if force or _stale(LIB, objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    print(build_lib(force="--force" in os.sys.argv, verbose=True))
