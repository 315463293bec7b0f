#!/usr/bin/env python3
"""Build libloom_hip.so (gfx950) from csrc/*.hip with hipcc, in-tree.

    python loomformer-paraplex_amd/build_lib.py [-j N]

Objects go to loomformer-paraplex_amd/_build/, the library to
loomformer-paraplex_amd/loom_amd/libloom_hip.so (loaded by loom_amd._lib), and
the host module of the per-token operators (csrc/host_ops.cpp, no device code)
to loom_amd/_host.so beside it.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
OUT = os.path.join(PKG, "loom_amd", "libloom_hip.so")
HOST_SRC = os.path.join(CSRC, "host_ops.cpp")
HOST_OUT = os.path.join(PKG, "loom_amd", "_host.so")
ARCH = "gfx950"

CFLAGS = [
    "-O3", "-fPIC", "-std=c++17", f"--offload-arch={ARCH}",
    # packed fp32 VALU ops are kept out of the code object on purpose
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-result",
]


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found (ROCm required to build libloom_hip.so)")
    return path


# per-source flags: the prefill attention keeps its MFMA accumulators in
# VGPRs (the default placed them in AGPRs, with a copy out and back for every
# online-softmax rescale; measured 122 -> 115 us per layer-chunk)
FILE_FLAGS = {"prefill.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}


def compile_one(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src).replace(".hip", ".o"))
    cmd = [hipcc(), *CFLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def torch_dir() -> str:
    """Where torch is installed (found without importing it)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("torch not found (its headers are needed for the host module)")
    return spec.submodule_search_locations[0]


def compile_host() -> str:
    obj = os.path.join(BUILD, "host_ops.o")
    inc = [os.path.join(torch_dir(), "include"), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           *(f"-isystem{d}" for d in inc), "-c", HOST_SRC, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {HOST_SRC}:\n{r.stdout}\n{r.stderr}")
    return obj


def link_host(obj: str) -> None:
    """The module against the library beside it and torch's own libraries (loaded by
    then: loom_amd imports torch first)."""
    tmp = HOST_OUT + ".tmp"
    cmd = ["g++", "-shared", obj, "-o", tmp, f"-L{os.path.dirname(OUT)}", "-l:libloom_hip.so",
           f"-L{os.path.join(torch_dir(), 'lib')}", "-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10",
           "-lamdhip64", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of the host module failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST_OUT)


def build(jobs: int = 8, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))
    with ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        host = ex.submit(compile_host)
        objs = list(ex.map(compile_one, srcs))
        host_obj = host.result()
    tmp = OUT + ".tmp"
    cmd = [hipcc(), "-shared", "-fPIC", f"--offload-arch={ARCH}", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OUT)
    link_host(host_obj)
    if verbose:
        print(f"built {OUT} from {len(srcs)} sources")
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=min(8, os.cpu_count() or 1))
    a = ap.parse_args()
    try:
        build(a.j, verbose=True)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
