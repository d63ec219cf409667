"""Build libkvint4.so (sm_100a) in-tree with nvcc.

    python kv-cache-triton_b200/build.py [--jobs N] [--force]

Each ``csrc/*.cu`` is compiled to an object under ``_build/`` and linked into
``kvint4/libkvint4.so`` next to the Python loader; ``csrc/binding.cpp`` becomes
``kvint4/_binding.so``, the torch-facing entry of the newer operators.  The CUDA runtime is linked
statically; the driver API entry point used for TMA descriptors is fetched at
run time, so the library loads on a machine without a GPU.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "kvint4", "libkvint4.so")
INCLUDE = os.path.join(ROOT, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xptxas", "-v", "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _stale(obj: str, src: str) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    deps = [src] + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    deps.append(os.path.join(INCLUDE, "kvint4.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def compile_one(src: str, force: bool) -> tuple[str, str]:
    obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
    if not force and not _stale(obj, src):
        return obj, ""
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    with open(obj + ".ptxas.txt", "w") as f:
        f.write(r.stderr)
    return obj, r.stderr


def build_binding(force: bool = False) -> str:
    """The Python extension: host code over torch's C++ headers and the library."""
    import sysconfig

    import torch
    src, out = os.path.join(CSRC, "binding.cpp"), os.path.join(HERE, "kvint4", "_binding.so")
    deps = [src, os.path.join(INCLUDE, "kvint4.h")]
    if not force and os.path.exists(out) and all(
            os.path.getmtime(d) <= os.path.getmtime(out) for d in deps):
        return out
    troot = os.path.dirname(torch.__file__)
    inc = [os.path.join(troot, "include"), os.path.join(troot, "include/torch/csrc/api/include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
           INCLUDE]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[x for d in inc for x in ("-isystem" if d != INCLUDE else "-I", d)], src,
           "-o", out + ".tmp", "-L", os.path.join(troot, "lib"), "-ltorch_python", "-ltorch_cpu",
           "-lc10", "-lc10_cuda", f"-Wl,-rpath,{os.path.join(troot, 'lib')}",
           "-L", os.path.join(HERE, "kvint4"), "-l:libkvint4.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"binding build failed:\n{r.stdout}\n{r.stderr}")
    os.replace(out + ".tmp", out)
    return out


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs) as ex:
        results = list(ex.map(lambda s: compile_one(s, force), srcs))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            if log:
                print(log)
    if force or not os.path.exists(OUT) or any(
            os.path.getmtime(o) > os.path.getmtime(OUT) for o in objs):
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", *objs,
               "-o", OUT + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(OUT + ".tmp", OUT)
    build_binding(force)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.jobs, verbose=a.verbose))
    sys.exit(0)
