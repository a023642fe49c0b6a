"""Build liblncc_sm100.so (the C-ABI CUDA library) in-tree for sm_100a, and libfused_lncc_torch.so, the torch operators of the
token blocks over it.

Usage: python fused-lncc_b200/build.py [--force] [--checked]

--checked builds the bounds-checked variant (LNCC_CHECKED=1) into liblncc_sm100_checked.so beside
the product library: every kernel access is range-checked and entry points report violations as
LNCC_ERR_CHECK (include/lncc.h, lncc_checked_build).

The reference builds a pybind torch extension for sm_70..sm_120 without sm_100
(reference setup.py:16-23,42-49). This builds a plain shared library for sm_100a only, with -O3
and -lineinfo and, like the reference, without --use_fast_math (the variance terms
Spp - Sp^2/n cancel and fast-math would cost accuracy). cudart is linked statically so that the
library carries its own runtime.
"""
import argparse
import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG_ROOT = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO_ROOT, "include")
LIB_DIR = os.path.join(PKG_ROOT, "fused_lncc")
LIB_NAME = "liblncc_sm100.so"
LIB_PATH = os.path.join(LIB_DIR, LIB_NAME)
CHECKED_LIB_PATH = os.path.join(LIB_DIR, "liblncc_sm100_checked.so")
TORCH_OPS_PATH = os.path.join(LIB_DIR, "libfused_lncc_torch.so")  # torch's view of the token-block operators
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = os.path.join(home, "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


OBJ_DIR = os.path.join(PKG_ROOT, "_build")


def sources(suffixes=(".cu", ".cuh", ".h")):
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(suffixes))


def _includes(path, seen=None):
    """The files of csrc/ and include/ that a source includes, itself among them."""
    seen = set() if seen is None else seen
    seen.add(path)
    with open(path) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    for name in names:
        for d in (CSRC, INCLUDE):
            dep = os.path.join(d, name)
            if os.path.exists(dep) and dep not in seen:
                _includes(dep, seen)
    return seen


def _stale(out):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    deps = sources() + [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd, out, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed building {out}:\n{r.stdout}\n{r.stderr}")


def build_library(force=False, checked=False, verbose=False, out=None):
    """Compile the library if it is missing or older than its sources; return its path. Each .cu file is an object of
    its own under _build/, compiled side by side and again only where it or what it includes is newer."""
    out = out or (CHECKED_LIB_PATH if checked else LIB_PATH)
    if not force and not _stale(out):
        return out
    objects = os.path.join(OBJ_DIR, "checked" if checked else "product")
    os.makedirs(objects, exist_ok=True)

    def compile_one(src):
        obj = os.path.join(objects, os.path.basename(src)[:-3] + ".o")
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(map(os.path.getmtime, _includes(src))):
            return obj
        cmd = [nvcc_path(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-I", INCLUDE, "-Xcompiler", "-fPIC",
               *(["-DLNCC_CHECKED=1"] if checked else []), "-c", "-o", f"{obj}.{os.getpid()}.tmp", src]
        _run(cmd, obj, verbose)
        os.replace(f"{obj}.{os.getpid()}.tmp", obj)
        return obj

    with ThreadPoolExecutor() as pool:
        built = list(pool.map(compile_one, sources((".cu",))))
    _run([nvcc_path(), *ARCH_FLAGS, "-Xcompiler", "-fPIC", "-shared", "-o", out + ".tmp", *built], out, verbose)
    os.replace(out + ".tmp", out)
    return out


def torch_mark():
    """The last bytes of libfused_lncc_torch.so: that it is whole, and the torch that it was compiled against, whose C++
    interface changes from version to version. fused_lncc/_native.py looks for them."""
    import torch
    return f"fused_lncc token blocks for torch {torch.__version__}, cxx11 abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}".encode()


def _ends_with(path, mark):
    if not os.path.exists(path) or os.path.getsize(path) < len(mark):
        return False
    with open(path, "rb") as f:
        f.seek(-len(mark), os.SEEK_END)
        return f.read() == mark


def build_torch_ops(force=False, verbose=False):
    """Compile csrc/torch_ops.cpp against the torch that is installed and the library beside it; return its path."""
    out, src = TORCH_OPS_PATH, os.path.join(CSRC, "torch_ops.cpp")
    lib = build_library(verbose=verbose)
    if not force and _ends_with(out, torch_mark()) and os.path.getmtime(out) >= max(map(os.path.getmtime, _includes(src))):
        return out
    import torch
    torch_dir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc_path())) or "/usr/local/cuda"
    includes = [INCLUDE, os.path.join(torch_dir, "include"),
                os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include"),
                sysconfig.get_paths()["include"]]
    # not $CXX: a compiler that links its own libstdc++ statically gives the library a second one beside torch's, and the
    # first number printed into an error message crashes
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in includes),
           "-o", out + ".tmp", src, f"-L{LIB_DIR}", f"-l:{os.path.basename(lib)}", f"-L{os.path.join(torch_dir, 'lib')}",
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    _run(cmd, out, verbose)
    with open(out + ".tmp", "ab") as f:
        f.write(torch_mark())
    os.replace(out + ".tmp", out)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--checked", action="store_true")
    args = ap.parse_args()
    p = build_library(force=args.force, checked=args.checked, verbose=True)
    print(p)
    if not args.checked:
        print(build_torch_ops(force=args.force, verbose=True))
    sys.exit(0)
