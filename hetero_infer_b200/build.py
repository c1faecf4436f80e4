"""Build the sm_100a shared library ``libhq4.so`` in-tree with nvcc.

The library is plain C ABI (``include/hq4.h``) over hand-written CUDA, without
torch headers.  Beside it, ``_hq4_torch`` (host code only, one file over torch's
headers) makes the paged operators' calls from tensors; the library builds and
works without it.  Both build without a GPU.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libhq4.so")
TORCH_SRC = os.path.join(CSRC, "hq4_torch.cpp")
TORCH_LIB = os.path.join(PKG, "_hq4_torch.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
              "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def headers():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def torch_version() -> str:
    """The installed torch's version, without importing it ('' where there is none)."""
    import importlib.metadata
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return ""


def built_for() -> str:
    """The torch version that _hq4_torch.so was built against, from the file beside it ('' for none)."""
    try:
        with open(TORCH_LIB + ".torch") as f:
            return f.read().strip()
    except OSError:
        return ""


def up_to_date(lib: str = LIB) -> bool:
    if not os.path.exists(lib):
        return False
    if lib == TORCH_LIB and built_for() != torch_version():  # torch's ABI is that of a version
        return False
    t = os.path.getmtime(lib)
    deps = [TORCH_SRC] if lib == TORCH_LIB else sources()
    return all(os.path.getmtime(f) <= t for f in deps + headers() + [__file__])


def torch_command():
    """The compile command of _hq4_torch."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    libdir = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = [f"-I{d}" for d in cpp_extension.include_paths() + [os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
                                                             sysconfig.get_paths()["include"], INCLUDE]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *inc, TORCH_SRC, "-o", TORCH_LIB + ".tmp",
            f"-L{libdir}", f"-Wl,-rpath,{libdir}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
            "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every csrc/*.cu into libhq4.so, and _hq4_torch.so (each skipped when up to date).

    libhq4.so needs nvcc alone.  Where _hq4_torch cannot be built (no torch, none of
    its headers, no host compiler) the reason goes to stderr, and the calls that
    need it (_lib.torch_calls) say that it is missing."""
    todo = [lib for lib in (LIB, TORCH_LIB) if force or not up_to_date(lib)]
    if not todo:
        return LIB
    import concurrent.futures
    import tempfile

    def run(cmd):
        out = subprocess.run(cmd, capture_output=True, text=True)
        if out.returncode != 0:
            raise RuntimeError("the build failed:\n" + " ".join(cmd) + "\n" + out.stdout + out.stderr)
        return out.stderr

    logs = []
    with tempfile.TemporaryDirectory() as tmp, \
            concurrent.futures.ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        binding = pool.submit(lambda: run(torch_command())) if TORCH_LIB in todo else None
        if LIB in todo:  # the files side by side, then one link
            objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in sources()]
            logs += pool.map(run, ([nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", s, "-o", o]
                                   for s, o in zip(sources(), objs)))
            run([nvcc(), *ARCH_FLAGS, "-shared", "-o", LIB + ".tmp", *objs])
            os.replace(LIB + ".tmp", LIB)
        if binding:
            try:
                logs.append(binding.result())
                os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
                with open(TORCH_LIB + ".torch", "w") as f:
                    f.write(torch_version() + "\n")
            except (ImportError, OSError, RuntimeError) as e:
                if os.path.exists(TORCH_LIB):  # it does not fit these sources
                    os.remove(TORCH_LIB)
                sys.stderr.write(f"{TORCH_LIB} was not built (libhq4.so is there without it): {e}\n")
    if verbose:
        sys.stdout.write("".join(logs))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
