"""Build librustorch_b200.so (sm_100a) in-tree with nvcc.

    python -m rustorch_b200.build [--force] [--verbose]

Each csrc/*.cu and csrc/*.cpp compiles to _build/*.o in parallel, then links into
rustorch_b200/librustorch_b200.so (NCCL is dlopen'ed at first use);
csrc/python/ops_module.cpp (the Python calls of the training and 8-bit operators)
compiles against torch's headers into rustorch_b200/_ops.so, and again when torch
or Python is another one (without torch only the library is built).  A source is
recompiled when it, any header or this file is newer than its object, and the
library is relinked when any object changed.  Objects and the library are stamped
with the time their compile started, so a file edited while a build runs is seen as
newer by the next build.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig
import time

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "librustorch_b200.so")
OPS_SRC = os.path.join(CSRC, "python", "ops_module.cpp")
OPS = os.path.join(PKG, "_ops.so")
OPS_STAMP = os.path.join(PKG, "_ops.torch")  # the torch and Python that OPS was built for
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
                     "-I" + os.path.join(ROOT, "include"), "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + [
        os.path.join(ROOT, "include", "rustorch_b200.h")]


def _obj(src: str) -> str:
    return os.path.join(BUILD, os.path.basename(src).rsplit(".", 1)[0] + ".o")


def _stale(src: str, newest_header: float) -> bool:
    obj = _obj(src)
    if not os.path.exists(obj):
        return True
    return os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header)


def _torch_tag():
    """The torch and Python that a module built now fits; None without torch.
    (torch is not imported: that takes seconds.)"""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return None
    version = runpy.run_path(os.path.join(os.path.dirname(spec.origin), "version.py"))["__version__"]
    return f"torch {version} {sysconfig.get_config_var('SOABI')}"


def ops_stale() -> bool:
    """The extension module is missing, older than its source or the C header, or
    made for another torch or Python."""
    if not (os.path.exists(OPS) and os.path.exists(OPS_STAMP)):
        return True
    with open(OPS_STAMP) as f:
        if f.read() != _torch_tag():
            return True
    t = os.path.getmtime(OPS)
    return any(os.path.getmtime(p) > t for p in (OPS_SRC, os.path.join(ROOT, "include",
                                                                       "rustorch_b200.h")))


def needs_build() -> bool:
    """The library is missing or older than a source or header (objects are
    not needed to use a library that is up to date)."""
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in _sources() + _headers() + [__file__])


def _compile(src: str, verbose: bool) -> str:
    obj = _obj(src)
    t0 = time.time()
    cmd = [_nvcc()] + NVCC_FLAGS + ["-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout or r.stderr):
        sys.stderr.write(r.stdout + r.stderr)
    os.utime(obj, (t0, t0))
    return obj


def _build_ops() -> None:
    import torch
    t0 = time.time()
    tdir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    inc = [os.path.join(tdir, "include"), os.path.join(tdir, "include", "torch", "csrc", "api",
                                                       "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    tmp = OPS + ".tmp"
    cmd = (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
           + ["-isystem" + i for i in inc] + [OPS_SRC, "-o", tmp, "-L" + PKG, "-lrustorch_b200",
                                              "-Wl,-rpath,$ORIGIN", "-L" + os.path.join(tdir, "lib"),
                                              "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"])
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {OPS_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OPS)
    os.utime(OPS, (t0, t0))
    with open(OPS_STAMP, "w") as f:
        f.write(_torch_tag())


def build(force: bool = False, verbose: bool = False) -> str:
    if force or needs_build():
        _build_lib(force, verbose)
    if _torch_tag() is None:
        sys.stderr.write("torch is not installed: the Python operators (_ops) are not built\n")
    elif force or ops_stale():
        _build_ops()
    return LIB


def _build_lib(force: bool, verbose: bool) -> None:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    hdr = max(os.path.getmtime(p) for p in _headers() + [__file__])  # (the flags are here)
    todo = [s for s in srcs if force or verbose or _stale(s, hdr)]
    if todo:
        with cf.ThreadPoolExecutor(max_workers=min(8, len(todo))) as ex:
            list(ex.map(lambda s: _compile(s, verbose), todo))
    objs = [_obj(s) for s in srcs]
    tmp = LIB + ".tmp"
    cmd = [_nvcc()] + ARCH + ["-shared", "-o", tmp] + objs + ["-lcudart_static",
                                                               "-lrt", "-ldl", "-lpthread"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    stamp = max(os.path.getmtime(o) for o in objs)
    os.utime(LIB, (stamp, stamp))


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
