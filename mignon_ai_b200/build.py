"""Builds libmignoncuda.so in-tree with nvcc for sm_100a (the only target)."""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmignoncuda.so")
UNITS = ("libmignoncuda", "libmignoncuda_kv")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v",
         "-ccbin", "/usr/bin/g++"]


def sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC))] + [
        os.path.join(os.path.dirname(HERE), "include", "mignon_cuda.h")]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    # the translation units side by side, then one link
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, u + ".o") for u in UNITS]
        jobs = [subprocess.Popen([NVCC, *FLAGS, "-c", "-o", o, os.path.join(CSRC, u + ".cu")], stdout=subprocess.PIPE,
                                 stderr=subprocess.STDOUT, text=True) for u, o in zip(UNITS, objs)]
        outs = [j.communicate()[0] for j in jobs]
        failed = any(j.returncode for j in jobs)
        if not failed:
            r = subprocess.run([NVCC, *FLAGS, "-shared", "-o", LIB, *objs], capture_output=True, text=True)
            outs.append(r.stdout + r.stderr)
            failed = r.returncode != 0
    if verbose or failed:
        sys.stderr.write("".join(outs))
    if failed:
        raise RuntimeError("nvcc failed building libmignoncuda.so")
    with open(os.path.join(HERE, "ptxas_info.txt"), "w") as f:
        f.write("".join(outs))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
