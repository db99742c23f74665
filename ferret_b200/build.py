"""Build the in-tree CUDA library ``ferret_b200/libferret_moe.so`` for sm_100a.

    python -m ferret_b200.build [--verbose] [--force]

Each ``csrc/*.cu`` is compiled by nvcc into ``_build/`` (in parallel) and the
objects are linked into one shared library with the CUDA runtime linked
statically, so the library loads on machines without a GPU driver (the
driver-API entry point the TMA descriptors need is resolved at run time
through the runtime).  ``kernel_result.cu`` becomes the benchmark binary
``ferret_b200/ferret_kernel_result`` linked against that library.
``csrc/host.cpp`` becomes the extension module ``ferret_b200/_host.so`` (g++
against the installed torch, linked to that library next to it), and again
when torch or Python changes; without a CUDA torch, g++ or Python's headers it is
left out, and the library and the C ABI are complete without it.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libferret_moe.so")
BIN = os.path.join(HERE, "ferret_kernel_result")
HOST = os.path.join(HERE, "_host.so")
HOST_FOR = os.path.join(HERE, "_host.for")      # what HOST was built against
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
          "--expt-relaxed-constexpr", "-I", INCLUDE]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build ferret_b200")
    return cand


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    return [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]


def _deps():
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != "host.cpp"] + _headers() + [
        os.path.join(HERE, "kernel_result.cu"), __file__]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def host_unavailable() -> str | None:
    """Why the extension module cannot be built here, or None."""
    torch = importlib.util.find_spec("torch")
    if torch is None or torch.origin is None:
        return "torch is not installed"
    if not os.path.exists(os.path.join(os.path.dirname(torch.origin), "lib", "libc10_cuda.so")):
        return "the installed torch has no CUDA"
    if not shutil.which("g++"):
        return "g++ was not found"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers are not installed"
    return None


def _host_for() -> str:
    try:
        torch_version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        import torch
        torch_version = torch.__version__
    return f"torch {torch_version}, {sys.implementation.cache_tag}"


def _host_stale() -> bool:
    if _stale(HOST, [os.path.join(CSRC, "host.cpp"), *_headers(), __file__]):
        return True
    try:
        with open(HOST_FOR) as f:
            return f.read() != _host_for()
    except OSError:
        return True


def build(verbose: bool = False, force: bool = False, ptxas_verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    missing = host_unavailable()
    library = force or any(_stale(t, _deps()) for t in (LIB, BIN))
    if library:
        build_library(srcs, verbose, ptxas_verbose)
    if missing is None:
        if force or _host_stale():
            build_host(verbose)
    elif library:
        print(f"ferret_b200: extension module not built ({missing}); the library is complete",
              file=sys.stderr)
    return LIB


def build_library(srcs, verbose: bool = False, ptxas_verbose: bool = False) -> None:
    """The shared library from its sources, and the benchmark binary."""
    cc = nvcc()
    extra = ["-Xptxas", "-v"] if ptxas_verbose else []

    def compile_one(src):
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        cmd = [cc, *ARCH, *CFLAGS, *extra, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        results = list(ex.map(compile_one, srcs))
    objs = [o for o, _ in results]
    if verbose or ptxas_verbose:
        for _, err in results:
            if err:
                print(err, file=sys.stderr)
    tmp = LIB + ".tmp"
    cmd = [cc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", *objs, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    build_kernel_result(cc, verbose)


def build_kernel_result(cc: str, verbose: bool = False) -> str:
    """The self-contained benchmark binary (KERNEL_RESULT lines), linked
    against the library next to it."""
    src = os.path.join(HERE, "kernel_result.cu")
    cmd = [cc, *ARCH, "-O2", "-std=c++17", src, "-o", BIN, "-L", HERE, "-lferret_moe",
           "-Xlinker", "-rpath,$ORIGIN", "-cudart", "static"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"kernel_result build failed:\n{r.stdout}\n{r.stderr}")
    return BIN


def build_host(verbose: bool = False) -> str:
    """The extension module of the operators' host side, linked against the
    library next to it and the installed torch."""
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    tmp = HOST + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", os.path.join(root, "include"),
           "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"),
           os.path.join(CSRC, "host.cpp"), "-o", tmp, "-L", HERE, "-lferret_moe",
           "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
           "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"host module build failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST)
    with open(HOST_FOR, "w") as f:
        f.write(_host_for())
    return HOST


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print ptxas register/smem usage")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force, ptxas_verbose=a.ptxas))


if __name__ == "__main__":
    main()
