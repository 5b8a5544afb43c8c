"""Build libnt_b200.so in-tree with nvcc for sm_100a (B200).

    python -m neural_textures_b200.build [--force] [--jobs N]

Each .cu under csrc/ compiles to an object in _build/ (in parallel), then one link step
produces neural_textures_b200/lib/libnt_b200.so; csrc/nt_torch.cpp (the texel layers' shortcut from torch
tensors to that library) becomes lib/nt_torch.so.  The build is incremental on file
modification times (any header change rebuilds everything).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libnt_b200.so")
TORCH_LIB = os.path.join(LIBDIR, "nt_torch.so")
NVCC = os.environ.get("NVCC", os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
         "-DNT_BUILD_LIBRARY"]


def _headers():
    return (glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
            + glob.glob(os.path.join(ROOT, "include", "neural_textures", "*.h")))


def _compile(src: str, obj: str, verbose_ptxas: bool) -> str:
    cmd = [NVCC] + ARCH + FLAGS + ["-c", src, "-o", obj]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def build(force: bool = False, jobs: int | None = None, verbose_ptxas: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_mtime = max([os.path.getmtime(h) for h in _headers()] + [os.path.getmtime(__file__)])
    todo = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_mtime):
            todo.append((s, o))
    logs = []
    if todo:
        with cf.ThreadPoolExecutor(max_workers=jobs or min(len(todo), os.cpu_count() or 4)) as ex:
            for log in ex.map(lambda so: _compile(so[0], so[1], verbose_ptxas), todo):
                logs.append(log)
    need_link = force or bool(todo) or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(
        os.path.getmtime(o) for o in objs)
    if need_link:
        tmp = LIB + ".tmp"
        cmd = [NVCC] + ARCH + ["-shared", "-o", tmp] + objs + ["-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if verbose_ptxas:
        sys.stderr.write("".join(logs))
    _build_torch(force)
    return LIB


def _build_torch(force: bool) -> None:
    src = os.path.join(CSRC, "nt_torch.cpp")
    needs = [src, os.path.join(ROOT, "include", "nt_capi.h"), __file__]
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) >= max(os.path.getmtime(n) for n in needs):
        return
    torch_dir = importlib.util.find_spec("torch").submodule_search_locations[0]  # without importing it
    cuda = os.path.dirname(os.path.dirname(NVCC))
    tmp = TORCH_LIB + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-I", os.path.join(ROOT, "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(torch_dir, "include"), "-I", os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(cuda, "include"), src, "-o", tmp, "-L", LIBDIR, "-l:libnt_b200.so", "-Wl,-rpath,$ORIGIN",
           "-L", os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cuda", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for nt_torch.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("--ptxas-verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(a.force, a.jobs, a.ptxas_verbose))


if __name__ == "__main__":
    main()
