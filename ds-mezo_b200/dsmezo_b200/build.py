"""Builds libdsmezo.so in-tree for sm_100a with nvcc.

    python -m dsmezo_b200.build        (from ds-mezo_b200/, or with it on sys.path)

Each source is compiled to its own object, side by side, then linked. No fast-math: the
Philox/Box-Muller draws must round exactly like torch's own build.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(HERE)
REPO = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
OBJ = os.path.join(PKG_ROOT, "_build")
OUT = os.path.join(HERE, "libdsmezo.so")
SOURCES = ["dsmz_api.cu", "dsmz_first_order.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found")
    return exe


def needs_build() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(INCLUDE, "dsmezo.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    flags = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
    jobs, objs = [], []
    for s in SOURCES:
        obj = os.path.join(OBJ, f"{os.path.splitext(s)[0]}.{os.getpid()}.o")
        cmd = [nvcc(), *flags, f"-I{INCLUDE}", f"-I{CSRC}", "-c", "-o", obj, os.path.join(CSRC, s)]
        if verbose:
            print(" ".join(cmd))
        jobs.append((cmd, subprocess.Popen(cmd)))
        objs.append(obj)
    try:
        codes = [(cmd, p.wait()) for cmd, p in jobs]
        for cmd, rc in codes:
            if rc != 0:
                raise subprocess.CalledProcessError(rc, cmd)
        tmp = f"{OUT}.{os.getpid()}.tmp"
        subprocess.run([nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs], check=True)
        os.replace(tmp, OUT)
    finally:
        for o in objs:
            if os.path.exists(o):
                os.remove(o)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
