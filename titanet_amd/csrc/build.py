#!/usr/bin/env python3
"""Build libtitanet_amd.so for gfx950 with hipcc (cross-compiles without a GPU).

    python titanet_amd/csrc/build.py [--force]

The library lands next to the package (titanet_amd/libtitanet_amd.so): it is git-ignored
but travels with the repo snapshot to the GPU box.
"""
import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
SOURCES = ["tn_api.hip", "tn_bwd.hip", "tn_mel.hip", "tn_optim.hip", "tn_int8.hip"]
# every header next to the sources feeds the rebuild digest (a stale .so must never ship: it travels prebuilt)
HEADERS = sorted(f for f in os.listdir(HERE) if f.endswith(".h")) + ["../../include/titanet_amd.h"]
OUT = os.path.join(PKG, "libtitanet_amd.so")
HOST_SOURCE, HOST_OUT = "tn_host.cpp", os.path.join(PKG, "_host.so")      # Python module over torch tensors, linked to the library
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics", "-Wall", "-Wno-unused-function",
         "-Wno-unused-variable",
         # ordinary float code becomes packed single-precision instructions at -O3 unless told otherwise; some of their forms are not
         # to be relied on, so no kernel here uses them (hipcc's host pass warns that it does not know the feature: harmless)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]



def _digest():
    h = hashlib.sha256()
    for f in SOURCES + HEADERS + [HOST_SOURCE, "build.py"]:
        path = os.path.join(HERE, f)
        if os.path.exists(path):
            with open(path, "rb") as fh:
                h.update(fh.read())
    return h.hexdigest()


def _build_host(verbose):
    import sysconfig

    import torch
    base = os.path.dirname(torch.__file__)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-I" + os.path.join(base, "include"), "-I" + os.path.join(base, "include", "torch", "csrc", "api", "include"),
           "-I" + os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"), "-I" + sysconfig.get_paths()["include"],
           os.path.join(HERE, HOST_SOURCE), "-o", HOST_OUT, "-L" + os.path.join(base, "lib"), "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu",
           "-ltorch_python", "-L" + PKG, "-l:" + os.path.basename(OUT), "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def build(force=False, verbose=True):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    stamp = os.path.join(HERE, ".build_stamp")
    dig = _digest()
    if not force and os.path.exists(OUT) and os.path.exists(HOST_OUT) and os.path.exists(stamp) and open(stamp).read().strip() == dig:
        return OUT
    objs = []

    def cc(src):
        obj = os.path.join(HERE, src.replace(".hip", ".o"))
        cmd = [hipcc] + FLAGS + ["-c", os.path.join(HERE, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=4) as ex:
        objs = list(ex.map(cc, SOURCES))
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    _build_host(verbose)
    with open(stamp, "w") as fh:
        fh.write(dig)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print("built", OUT)
